// Leaky attention: linear attention with a decay for each head.  leaky_attn.h
// has the recurrence, its gradients and how one kernel serves all of them.
//
// This file: the entry points, the kernel on the fp32 pipe, the joining of time
// segments, the sum of shared heads' gradients and the single-token step.
//
// Chunked form, C tokens at a time with the state S before the chunk:
//   o_i = p * sum_{j <= i} b^(i-j) (q_i . k_j) v_j + c * b^(i+1) S^T q_i
//   S  <- b^C S + sum_j b^(C-1-j) k_j v_j^T
// Operations a token and head: C (dq + dv) / 2 within the chunk (causal half) and
// 2 dq dv for the state, against (2 dq + 2 dv) elements read and written.
//
// Time segments: a head is a chain over its chunks.  Where B * H chains cannot
// fill the GPU, time is cut into segments: a first launch forms each segment's
// own end state from zero, k_attn_join turns them into starting states
// (start[u + 1] = b^n start[u] + own[u]), and the main launch runs all segments
// at once.
#include <algorithm>

#include "leaky_attn.h"
#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"

namespace lifb {

namespace {

constexpr int kAtC = 32;         // tokens of a chunk
constexpr int kAtThreads = 128;
constexpr int kAtTile = 64;      // columns of v of one block
constexpr int kAtSV = kAtTile + 4, kAtSP = kAtC + 4;  // padded row lengths in shared memory
constexpr int kAtSms = 148;

}  // namespace

// Rows [t0, t0 + kAtC) of a [tokens, d] operand into dst[row][col], zeros past
// n rows and d columns.  W4: four elements at a time.
template <typename T, bool W4>
__device__ __forceinline__ void attn_load(float *dst, int ld, const T *src, int64_t st, int n, int d, int cols)
{
    if (W4) {
        const int per = cols / 4;
        for (int i = threadIdx.x; i < kAtC * per; i += kAtThreads) {
            const int r = i / per, c = (i - r * per) * 4;
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < n && c < d) load_f32(src + r * st + c, x);
            *reinterpret_cast<float4 *>(dst + r * ld + c) = make_float4(x[0], x[1], x[2], x[3]);
        }
    } else {
        for (int i = threadIdx.x; i < kAtC * cols; i += kAtThreads) {
            const int r = i / cols, c = i - r * cols;
            dst[r * ld + c] = r < n && c < d ? to_f32(src[r * st + c]) : 0.0f;
        }
    }
}

// One block: one (pass, sequence, head, time segment) and kAtTile columns of v.
// 128 threads as 8 x 16: 4 rows x 4 columns of a [32, 64] output each.  The
// state lives in shared memory in fp32.  Bound by the fp32 pipe: a chunk is 32 (dq (2 64
// + 16) + 64 16) multiply-adds a block at 128 a cycle (B 64, T 1024, H 4, 64 x 64 forward:
// 220 us of them, 465 us measured).  What comes here is what the tensor-core kernels do
// not take: widths, strides or addresses that are not multiples of 16 bytes.
template <typename T, bool W4>
__global__ void __launch_bounds__(kAtThreads) k_attn_simt(const __grid_constant__ AttnArgs a, int state_only)
{
    const AttnPass &p = a.p[blockIdx.z];
    const int v0 = blockIdx.y * kAtTile;
    if (v0 >= p.dv) return;
    const int64_t bh = blockIdx.x / a.nseg;
    const int u = (int)(blockIdx.x - bh * a.nseg);  // in the order of the pass
    if (state_only && u == a.nseg - 1) return;      // nothing starts from the last one
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int dv = min(kAtTile, p.dv - v0), dq = p.dq, dq4 = (dq + 3) & ~3, ldq = dq4 + 4;
    const int64_t len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[h];

    extern __shared__ float4 at_smem4[];
    float *Q = reinterpret_cast<float *>(at_smem4), *K = Q + kAtC * ldq, *V = K + kAtC * ldq, *P = V + kAtC * kAtSV,
          *S = P + kAtC * kAtSP;
    __shared__ float wi[kAtC], wk[kAtC], pw[kAtC];
    const int tid = threadIdx.x, ti = tid >> 4, tj = tid & 15;

    const T *q = (const T *)p.q + b * p.qs[0] + (h / p.qg) * p.qs[2];
    const T *k = (const T *)p.k + b * p.ks[0] + (h / p.kg) * p.ks[2];
    const T *v = (const T *)p.v + b * p.vs[0] + (h / p.vg) * p.vs[2] + v0;
    char *o = (char *)p.o + (b * p.os[0] + h * p.os[2] + v0) * (p.o_f32 ? 4 : (int)sizeof(T));

    // the segment's starting state
    const int64_t mat = (int64_t)p.dq * p.dv;
    const float *s_in = nullptr;
    int64_t row = p.s_row, col = p.s_col;
    if (!state_only) {
        if (u == 0) {
            if (p.s_in) s_in = p.s_in + bh * mat;
        } else {
            s_in = p.seg + (bh * (a.nseg + 1) + u) * mat;
            row = p.dv;
            col = 1;
        }
    }
    for (int i = tid; i < dq4 * kAtTile; i += kAtThreads) {
        const int r = i / kAtTile, c = i % kAtTile;
        S[r * kAtSV + c] = s_in && r < dq && c < dv ? s_in[r * row + (v0 + c) * col] : 0.0f;
    }
    const DecayFactor full(ld, kAtC);
    if (tid < kAtC) pw[tid] = decay_pow(ld, (float)tid);

    const int64_t seg = p.rev ? a.nseg - 1 - u : u;  // in time
    const int64_t s0 = seg * a.seg_tokens, s1 = min(a.T, s0 + a.seg_tokens);
    const int64_t chunks = s1 > s0 ? (s1 - s0 + kAtC - 1) / kAtC : 0;
    for (int64_t cc = 0; cc < chunks; cc++) {
        const int64_t t0 = s0 + (p.rev ? chunks - 1 - cc : cc) * kAtC;
        const int rows = (int)min((int64_t)kAtC, s1 - t0);
        const int n = (int)max((int64_t)0, min((int64_t)rows, len - t0));
        __syncthreads();  // the last chunk's readers are done
        if (n > 0) {
            if (!state_only) attn_load<T, W4>(Q, ldq, q + t0 * p.qs[1], p.qs[1], n, dq, dq4);
            attn_load<T, W4>(K, ldq, k + t0 * p.ks[1], p.ks[1], n, dq, dq4);
            attn_load<T, W4>(V, kAtSV, v + t0 * p.vs[1], p.vs[1], n, dv, kAtTile);
            if (tid < kAtC) {
                const int r = p.rev ? n - 1 - tid : tid;  // tokens of the chunk seen before this one
                wi[tid] = tid < n ? p.i_scale * decay_pow(ld, (float)(r + 1 - p.shift)) : 0.0f;
                wk[tid] = tid < n ? p.w_scale * decay_pow(ld, (float)(n - 1 - r + p.shift)) : 0.0f;
            }
        }
        __syncthreads();
        float acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = 0.0f;
        if (n > 0 && !state_only) {
            // P = p_scale * decay * Q K^T: rows 4 ti + i, columns tj and tj + 16
            float s[4][2] = {};
            for (int c = 0; c < dq4; c += 4) {
                float4 x[4], y[2];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4 *>(Q + (4 * ti + i) * ldq + c);
#pragma unroll
                for (int j = 0; j < 2; j++) y[j] = *reinterpret_cast<const float4 *>(K + (tj + 16 * j) * ldq + c);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        s[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int r = 4 * ti + i, c = tj + 16 * j, d = p.rev ? c - r : r - c;
                    P[r * kAtSP + c] = d >= 0 ? p.p_scale * pw[d] * s[i][j] : 0.0f;
                }
            // the carried term: Q S, then the row's weight
            for (int c = 0; c < dq4; c += 4) {
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4 *>(Q + (4 * ti + i) * ldq + c);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float4 y = *reinterpret_cast<const float4 *>(S + (c + e) * kAtSV + 4 * tj);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float xe = e == 0 ? x[i].x : e == 1 ? x[i].y : e == 2 ? x[i].z : x[i].w;
                        acc[i][0] += xe * y.x;
                        acc[i][1] += xe * y.y;
                        acc[i][2] += xe * y.z;
                        acc[i][3] += xe * y.w;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] *= wi[4 * ti + i];
        }
        __syncthreads();  // P is written, S read
        if (n > 0 && !state_only) {
            for (int c = 0; c < kAtC; c += 4) {
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const float4 *>(P + (4 * ti + i) * kAtSP + c);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float4 y = *reinterpret_cast<const float4 *>(V + (c + e) * kAtSV + 4 * tj);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float xe = e == 0 ? x[i].x : e == 1 ? x[i].y : e == 2 ? x[i].z : x[i].w;
                        acc[i][0] += xe * y.x;
                        acc[i][1] += xe * y.y;
                        acc[i][2] += xe * y.z;
                        acc[i][3] += xe * y.w;
                    }
                }
            }
        }
        if (!state_only) {  // rows past the sequence's end are zero
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 4 * ti + i;
                if (r >= rows) continue;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int c = 4 * tj + j;
                    if (c >= dv) continue;
                    const int64_t at = (t0 + r) * p.os[1] + c;
                    if (p.o_f32) ((float *)o)[at] = acc[i][j];
                    else ((T *)o)[at] = from_f32<T>(acc[i][j]);
                }
            }
        }
        if (n > 0) {
            // S = b^n S + K^T diag(wk) V: rows 4 ti + 32 m, columns 4 tj
            const DecayFactor bn = n == kAtC ? full : DecayFactor(ld, n);
            float st[4][4][4];
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const int r = 4 * ti + 32 * m;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 y = r < dq4 ? *reinterpret_cast<const float4 *>(S + (r + i) * kAtSV + 4 * tj)
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    st[m][i][0] = bn.times(y.x);
                    st[m][i][1] = bn.times(y.y);
                    st[m][i][2] = bn.times(y.z);
                    st[m][i][3] = bn.times(y.w);
                }
            }
            for (int j = 0; j < n; j++) {
                const float w = wk[j];
                float4 y = *reinterpret_cast<const float4 *>(V + j * kAtSV + 4 * tj);
                y.x *= w;
                y.y *= w;
                y.z *= w;
                y.w *= w;
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    const int r = 4 * ti + 32 * m;
                    if (r >= dq4) break;
                    const float4 x = *reinterpret_cast<const float4 *>(K + j * ldq + r);
                    const float xe[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        st[m][i][0] += xe[i] * y.x;
                        st[m][i][1] += xe[i] * y.y;
                        st[m][i][2] += xe[i] * y.z;
                        st[m][i][3] += xe[i] * y.w;
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const int r = 4 * ti + 32 * m;
                if (r >= dq4) break;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<float4 *>(S + (r + i) * kAtSV + 4 * tj) =
                        make_float4(st[m][i][0], st[m][i][1], st[m][i][2], st[m][i][3]);
            }
        }
    }
    __syncthreads();
    float *s_out = nullptr;
    if (state_only) {
        s_out = p.seg + (bh * (a.nseg + 1) + u + 1) * mat;
        row = p.dv;
        col = 1;
    } else if (u == a.nseg - 1 && p.s_out) {
        s_out = p.s_out + bh * mat;
        row = p.s_row;
        col = p.s_col;
    }
    if (s_out)
        for (int i = tid; i < dq * kAtTile; i += kAtThreads) {
            const int r = i / kAtTile, c = i % kAtTile;
            if (c < dv) s_out[r * row + (v0 + c) * col] = S[r * kAtSV + c];
        }
}

// Segments' own end states to starting states: seg[u] += b^n(u - 1) seg[u - 1],
// seg[0] the pass's initial state; `finish`: the final state from the last one too.
// One element a thread, in the order of the pass.
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ AttnArgs a, int finish)
{
    const AttnPass &p = a.p[blockIdx.z];
    const int64_t mat = (int64_t)p.dq * p.dv, bh = blockIdx.y, e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= mat) return;
    const int64_t b = bh / a.H, len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[bh - b * a.H];
    const DecayFactor full(ld, a.seg_tokens);
    const int64_t r = e / p.dv, c = e - r * p.dv;
    float s = p.s_in ? p.s_in[bh * mat + r * p.s_row + c * p.s_col] : 0.0f;
    float *at = p.seg + bh * (a.nseg + 1) * mat + e;
    const int last = a.nseg + (finish && p.s_out);
    for (int u0 = 1; u0 < last; u0 += 8) {  // eight loads in flight
        float own[8];
#pragma unroll
        for (int j = 0; j < 8; j++) own[j] = u0 + j < last ? at[(u0 + j) * mat] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int u = u0 + j;
            if (u >= last) break;
            const int64_t seg = p.rev ? a.nseg - u : u - 1;  // in time, the one before
            const int64_t s0 = seg * a.seg_tokens, s1 = min(a.T, s0 + a.seg_tokens);
            const int64_t n = max((int64_t)0, min(s1, len) - s0);
            s = (n == a.seg_tokens ? full : DecayFactor(ld, n)).times(s) + own[j];
            if (u == a.nseg) p.s_out[bh * mat + r * p.s_row + c * p.s_col] = s;
            else at[u * mat] = s;
        }
    }
}

// Gradients of shared heads: out[.., hk, :] = the sum of part[.., hk * g + i, :]
// over i < g, in order (fp32 parts, rounded once).
template <typename T>
__global__ void __launch_bounds__(256) k_attn_group(const float *__restrict__ part, T *__restrict__ out, int64_t rows,
                                                    int g, int d)
{
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * d; i += step) {
        const int64_t r = i / d, c = i - r * d;
        float s = 0.0f;
        for (int j = 0; j < g; j++) s += part[(r * g + j) * d + c];
        out[i] = from_f32<T>(s);
    }
}

// A state's elements, read once and written once: not kept in the caches.
template <int VEC>
__device__ __forceinline__ void load_once(const float *p, float (&x)[VEC])
{
    if constexpr (VEC == 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4 *>(p));
        x[0] = f.x;
        x[1] = f.y;
        x[2] = f.z;
        x[3] = f.w;
    } else {
        x[0] = __ldcs(p);
    }
}
template <int VEC>
__device__ __forceinline__ void store_once(float *p, const float (&x)[VEC])
{
    if constexpr (VEC == 4) __stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
    else __stcs(p, x[0]);
}

// One token: S = b S + k v^T in place, o = scale * S^T q.  A block has one
// (sequence, head) and CV * VEC columns of the state; its threads are CV columns
// (VEC elements each) by row groups that walk the rows, and the groups' sums of
// q_r S_r are added at the end.  Bound by memory: the state is read and written
// once, 8 dk dv bytes.  What it takes is enough bytes in flight: eight rows a thread
// are on their way before q and k are (190 sequences of 16 heads of 128 x 128: 80 us
// with the rows after them, 68 us so, 62 us at the copy rate), and blocks of 128
// threads, 16 vectors wide, so that heads of 64 x 64 do too (512 x 16 of them: 60 us
// with 256 threads, 48 us so, floor 42 us).
template <typename T, int VEC>
__global__ void __launch_bounds__(kAtThreads)
    k_attn_step(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ o,
                const float *__restrict__ log_decay, float *__restrict__ state, const int32_t *__restrict__ slots,
                int64_t n_slots, int H, int group, int dk, int dv, int cv, int64_t q_b, int64_t q_h, int64_t k_b,
                int64_t k_h, int64_t v_b, int64_t v_h, int64_t s_slot, int64_t s_h, float scale)
{
    __shared__ float sq[kAttnMaxDim], sk[kAttnMaxDim];
    __shared__ float part[kAtThreads * VEC];
    const int64_t b = blockIdx.x / H, h = blockIdx.x - b * H;
    const int tid = threadIdx.x, groups = blockDim.x / cv, rg = tid / cv;
    const int c = (blockIdx.y * cv + tid % cv) * VEC;
    const int64_t slot = slots ? slots[b] : b;
    const bool live = slot >= 0 && slot < n_slots;
    if (!live) {  // uniform over the block
        if (rg == 0 && c < dv) {
            float z[VEC] = {};
            store_f32(o + (b * H + h) * dv + c, z);
        }
        return;
    }
    for (int i = tid; i < dk; i += blockDim.x) {
        sq[i] = to_f32(q[b * q_b + h * q_h + i]) * scale;
        sk[i] = to_f32(k[b * k_b + (h / group) * k_h + i]);
    }
    const float beta = expf(log_decay[h]);
    float x[VEC], acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) x[e] = acc[e] = 0.0f;
    float *st = state + slot * s_slot + h * s_h + c;
    const bool in = c < dv && rg < groups;
    // rows rg, rg + groups, ..., U of them in flight; the first ones before q and k are there
    constexpr int U = 8;
    float y[U][VEC];
    auto load = [&](int r0) {
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int r = r0 + j * groups;
            if (in && r < dk) load_once(st + (int64_t)r * dv, y[j]);
        }
    };
    load(rg);
    if (in) load_f32(v + b * v_b + (h / group) * v_h + c, x);
    __syncthreads();
    for (int r0 = rg; r0 < dk; r0 += U * groups) {
        if (r0 != rg) load(r0);
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int r = r0 + j * groups;
            if (!in || r >= dk) break;
            const float kr = sk[r], qr = sq[r];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                y[j][e] = beta * y[j][e] + kr * x[e];
                acc[e] += qr * y[j][e];
            }
            store_once(st + (int64_t)r * dv, y[j]);
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; e++) part[tid * VEC + e] = acc[e];
    __syncthreads();
    if (rg == 0 && c < dv) {
        for (int i = 1; i < groups; i++)
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[e] += part[(i * cv + tid) * VEC + e];
        store_f32(o + (b * H + h) * dv + c, acc);
    }
}

namespace {

bool four_wide(const void *p, const int64_t *st, int d, int elem)
{
    return (uintptr_t)p % (4 * elem) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0 && d % 4 == 0;
}

template <typename T, bool W4>
bool launch_simt(const AttnArgs &a, int passes, bool state_only, cudaStream_t s)
{
    int dq = 0, dv = 0;
    for (int i = 0; i < passes; i++) {
        dq = std::max(dq, (a.p[i].dq + 3) & ~3);
        dv = std::max(dv, a.p[i].dv);
    }
    auto bytes = [](int dq) {  // 80 KB at dq = 128
        return ((size_t)2 * kAtC * (dq + 4) + (size_t)kAtC * kAtSV + (size_t)kAtC * kAtSP + (size_t)dq * kAtSV) * 4;
    };
    const size_t smem = bytes(dq);
    // the kernel's limit is the most that any width takes: it is one for all threads, and a
    // call's own size could lower it under another's launch
    auto kern = k_attn_simt<T, W4>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes(kAttnMaxDim)) != cudaSuccess)
        return false;
    count_launches(1);
    kern<<<dim3((unsigned)(a.B * a.H * a.nseg), (unsigned)((dv + kAtTile - 1) / kAtTile), (unsigned)passes), kAtThreads,
           smem, s>>>(a, state_only);
    return true;
}

}  // namespace

bool attn_simt(const AttnArgs &a, int passes, int dtype, bool state_only, cudaStream_t s)
{
    const int elem = (int)dtype_bytes(dtype);
    bool w4 = true;
    for (int i = 0; i < passes; i++) {
        const AttnPass &p = a.p[i];
        w4 = w4 && four_wide(p.q, p.qs, p.dq, elem) && four_wide(p.k, p.ks, p.dq, elem) &&
             four_wide(p.v, p.vs, p.dv, elem);
    }
    if (dtype == LIFB_F32)
        return w4 ? launch_simt<float, true>(a, passes, state_only, s) : launch_simt<float, false>(a, passes, state_only, s);
    return w4 ? launch_simt<__nv_bfloat16, true>(a, passes, state_only, s)
              : launch_simt<__nv_bfloat16, false>(a, passes, state_only, s);
}

namespace {

int at_fail(int status, const char *what, const char *why)
{
    char msg[200];
    snprintf(msg, sizeof msg, "%s: %s", what, why);
    set_last_error(msg);
    return status;
}

struct Split {
    int nseg;
    int64_t seg_tokens;
};

// Time segments for `chains` chains of T tokens, `room` blocks resident on the
// GPU at once.  A split costs a second read of k and v for the segments' own
// states (about half a pass), so it is taken when the waves of whole chains
// take longer than the waves of segments and that pass together.
Split split_time(int64_t chains, int64_t T, int64_t room)
{
    Split best = {1, (T + kAttnSegGrain - 1) / kAttnSegGrain * kAttnSegGrain};
    const int64_t grains = (T + kAttnSegGrain - 1) / kAttnSegGrain;
    if (chains == 0 || grains < 2) return best;
    double best_t = (double)((chains + room - 1) / room) * grains;
    for (int64_t want = 2; want <= std::min<int64_t>(grains, 64); want++) {
        const int64_t per = (grains + want - 1) / want, n = (grains + per - 1) / per;
        // + 1: the state's way into and out of a segment, and the joining launch
        const double t = (double)((chains * n + room - 1) / room) * (per + 1.0) +
                         0.5 * ((chains * (n - 1) + room - 1) / room) * (per + 1.0) + 2.0;
        if (t < best_t * 0.95) {
            best_t = t;
            best = {(int)n, per * kAttnSegGrain};
        }
    }
    return best;
}

// Blocks that the GPU holds at once, of the kernel that the type and widths point to.
int64_t attn_room(int64_t dq, int64_t dv, int dtype)
{
    if (dtype == LIFB_BF16 && dq % 8 == 0 && dv % 8 == 0) return kAtSms;
    if (dtype == LIFB_F32 && dq % 4 == 0 && dv % 4 == 0) return kAtSms;
    return kAtSms * 2 / std::max<int64_t>(1, (dv + kAtTile - 1) / kAtTile);
}

struct AttnWs {
    float *seg[kAttnMaxPasses];
    float *part[2];  // dk, dv of each query head, where heads are shared
    size_t bytes;
};

AttnWs carve(void *base, const lifb_leaky_attn &p, bool bwd, const Split &sp)
{
    AttnWs w = {};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        float *r = (float *)((char *)base + at);
        at += (bytes + 255) & ~(size_t)255;
        return r;
    };
    const size_t mat = (size_t)p.B * p.H * p.Dk * p.Dv * 4;
    // one segment: room for the final state of a pass that returns one
    for (int i = 0; i < (bwd ? 3 : 1); i++)
        if (sp.nseg > 1 || (p.dtype == LIFB_BF16 && (!bwd || i == 2))) w.seg[i] = take(mat * (sp.nseg + 1));
    if (bwd && p.Hk != p.H) {
        w.part[0] = take((size_t)p.B * p.T * p.H * p.Dk * 4);
        w.part[1] = take((size_t)p.B * p.T * p.H * p.Dv * 4);
    }
    w.bytes = at;
    return w;
}

Split split_of(const lifb_leaky_attn &p, bool bwd)
{
    // chains of one launch: passes, and in fp32 the parts of their widths
    int64_t k = 1, v = 1;
    if (p.dtype == LIFB_F32) k = (p.Dk + kT32W - 1) / kT32W, v = (p.Dv + kT32W - 1) / kT32W;
    return split_time(p.B * p.H * (bwd ? 2 * k + v : v), p.T, attn_room(p.Dk, p.Dv, p.dtype));
}

int at_check(const char *what, const lifb_leaky_attn *p)
{
    if (!p) return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null arguments");
    if (p->B < 0 || p->T < 0 || p->H < 0 || p->Hk < 0 || p->Dk < 0 || p->Dv < 0)
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "negative shape");
    if (p->dtype != LIFB_F32 && p->dtype != LIFB_BF16)
        return at_fail(LIFB_ERR_UNSUPPORTED, what, "q, k and v are fp32 or bf16");
    if (p->H > 0 && (p->Hk <= 0 || p->H % p->Hk))
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "H must be a multiple of Hk");
    if (p->Dk > kAttnMaxDim || p->Dv > kAttnMaxDim)
        return at_fail(LIFB_ERR_UNSUPPORTED, what, "head widths up to 128");
    if (p->T >= (int64_t(1) << 31) - 256 || p->B * p->H >= (int64_t(1) << 16))
        return at_fail(LIFB_ERR_UNSUPPORTED, what, "needs T < 2^31 - 256 and B * H < 2^16");
    return LIFB_OK;
}

bool run_passes(AttnArgs &a, int passes, int dtype, cudaStream_t s)
{
    a.passes = passes;
    const bool tc = attn_tc_applies(a, passes, dtype), tc32 = attn_tc32_applies(a, passes, dtype);
    // on the tensor cores a returned state comes from the state's own kernel, except where
    // the main one has it at hand
    bool finish = false;
    if (tc)
        for (int i = 0; i < passes; i++)
            finish = finish || (a.p[i].s_out && (a.nseg > 1 || !attn_tc_returns_state(a.p[i].dq, a.p[i].dv)));
    if (a.nseg > 1 || finish) {
        const bool ok = tc     ? attn_state(a, passes, finish, s)
                        : tc32 ? attn_tc32(a, passes, true, s)
                               : attn_simt(a, passes, dtype, true, s);
        if (!ok) return false;
        int64_t mat = 0;
        for (int i = 0; i < passes; i++) mat = std::max<int64_t>(mat, (int64_t)a.p[i].dq * a.p[i].dv);
        count_launches(1);
        k_attn_join<<<dim3((unsigned)((mat + 255) / 256), (unsigned)(a.B * a.H), (unsigned)passes), 256, 0, s>>>(a,
                                                                                                           finish);
        if (finish)
            for (int i = 0; i < passes; i++) a.p[i].s_out = nullptr;
    }
    return tc ? attn_tc(a, passes, s) : tc32 ? attn_tc32(a, passes, false, s) : attn_simt(a, passes, dtype, false, s);
}

void strides_of(int64_t (&st)[3], const int64_t *from) { st[0] = from[0], st[1] = from[1], st[2] = from[2]; }

void dense_strides(int64_t (&st)[3], int64_t T, int64_t H, int64_t D) { st[0] = T * H * D, st[1] = H * D, st[2] = D; }

}  // namespace

}  // namespace lifb

extern "C" size_t lifb_leaky_attn_workspace_bytes(const lifb_leaky_attn *p, int backward)
{
    using namespace lifb;
    if (at_check("lifb_leaky_attn_workspace_bytes", p)) return 0;
    if (p->B == 0 || p->T == 0 || p->H == 0 || p->Dk == 0 || p->Dv == 0) return 0;
    return carve(nullptr, *p, backward != 0, split_of(*p, backward != 0)).bytes;
}

extern "C" int lifb_leaky_attn_fwd(const lifb_leaky_attn *p, void *o, float *state_out, void *workspace,
                                   size_t workspace_bytes, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_leaky_attn_fwd");
    const char *what = "lifb_leaky_attn_fwd";
    if (int st = at_check(what, p)) return st;
    cudaStream_t s = (cudaStream_t)stream;
    const size_t state_bytes = (size_t)p->B * p->H * p->Dk * p->Dv * 4, o_bytes = (size_t)p->B * p->T * p->H * p->Dv * dtype_bytes(p->dtype);
    if (p->B == 0 || p->H == 0 || p->Dv == 0) return LIFB_OK;
    if ((p->T > 0 && !o) || !p->log_decay) return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    if (p->T == 0 || p->Dk == 0) {  // no token: the state stays; no key: nothing is stored or read
        bool ok = true;
        if (o_bytes) ok = cudaMemsetAsync(o, 0, o_bytes, s) == cudaSuccess;
        if (state_out && state_bytes)
            ok = ok && (p->state ? cudaMemcpyAsync(state_out, p->state, state_bytes, cudaMemcpyDeviceToDevice, s)
                                 : cudaMemsetAsync(state_out, 0, state_bytes, s)) == cudaSuccess;
        return ok ? LIFB_OK : at_fail(LIFB_ERR_CUDA, what, "memset or copy failed");
    }
    if (!p->q || !p->k || !p->v) return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    const Split sp = split_of(*p, false);
    const AttnWs w = carve(workspace, *p, false, sp);
    if (w.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < w.bytes))
        return at_fail(LIFB_ERR_WORKSPACE, what, "workspace missing, misaligned or too small");
    AttnArgs a = {};
    a.log_decay = p->log_decay;
    a.lengths = p->lengths;
    a.B = p->B, a.T = p->T, a.H = p->H;
    a.nseg = sp.nseg;
    a.seg_tokens = sp.seg_tokens;
    const int g = (int)(p->H / p->Hk);
    AttnPass &f = a.p[0];
    f.q = p->q, f.k = p->k, f.v = p->v, f.o = o;
    strides_of(f.qs, p->q_strides);
    strides_of(f.ks, p->k_strides);
    strides_of(f.vs, p->v_strides);
    dense_strides(f.os, p->T, p->H, p->Dv);
    f.qg = 1, f.kg = f.vg = g;
    f.dq = (int)p->Dk, f.dv = (int)p->Dv;
    f.s_in = p->state, f.s_out = state_out, f.s_row = p->Dv, f.s_col = 1;
    f.p_scale = f.i_scale = p->scale, f.w_scale = 1.0f;
    f.seg = w.seg[0];
    if (!run_passes(a, 1, p->dtype, s) || cudaGetLastError() != cudaSuccess)
        return at_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}

extern "C" int lifb_leaky_attn_bwd(const lifb_leaky_attn *p, const void *d_o, const int64_t *d_o_strides,
                                   const float *dstate_out, void *dq, void *dk, void *dv, float *dstate,
                                   void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_leaky_attn_bwd");
    const char *what = "lifb_leaky_attn_bwd";
    if (int st = at_check(what, p)) return st;
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t e = dtype_bytes(p->dtype);
    if (p->B == 0 || p->H == 0) return LIFB_OK;
    if (p->T == 0 || p->Dk == 0 || p->Dv == 0) {
        bool ok = true;
        auto zero = [&](void *x, int64_t heads, int64_t d) {
            const size_t nb = (size_t)p->B * p->T * heads * d * e;
            if (nb) ok = ok && x && cudaMemsetAsync(x, 0, nb, s) == cudaSuccess;
        };
        zero(dq, p->H, p->Dk);
        zero(dk, p->Hk, p->Dk);
        zero(dv, p->Hk, p->Dv);
        const size_t nb = (size_t)p->B * p->H * p->Dk * p->Dv * 4;
        if (dstate && nb)
            ok = ok && (dstate_out ? cudaMemcpyAsync(dstate, dstate_out, nb, cudaMemcpyDeviceToDevice, s)
                                   : cudaMemsetAsync(dstate, 0, nb, s)) == cudaSuccess;
        return ok ? LIFB_OK : at_fail(LIFB_ERR_CUDA, what, "memset or copy failed");
    }
    if (!p->q || !p->k || !p->v || !p->log_decay || !d_o || !d_o_strides || !dq || !dk || !dv)
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    const Split sp = split_of(*p, true);
    const AttnWs w = carve(workspace, *p, true, sp);
    if (w.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < w.bytes))
        return at_fail(LIFB_ERR_WORKSPACE, what, "workspace missing, misaligned or too small");
    AttnArgs a = {};
    a.log_decay = p->log_decay;
    a.lengths = p->lengths;
    a.B = p->B, a.T = p->T, a.H = p->H;
    a.nseg = sp.nseg;
    a.seg_tokens = sp.seg_tokens;
    const int g = (int)(p->H / p->Hk), dK = (int)p->Dk, dV = (int)p->Dv;
    // dq: forward on (do, v, k), the state transposed
    AttnPass &x = a.p[0];
    x.q = d_o, x.k = p->v, x.v = p->k, x.o = dq;
    strides_of(x.qs, d_o_strides);
    strides_of(x.ks, p->v_strides);
    strides_of(x.vs, p->k_strides);
    dense_strides(x.os, p->T, p->H, p->Dk);
    x.qg = 1, x.kg = x.vg = g;
    x.dq = dV, x.dv = dK;
    x.s_in = p->state, x.s_row = 1, x.s_col = dV;
    x.p_scale = x.i_scale = p->scale, x.w_scale = 1.0f;
    x.seg = w.seg[0];
    // dk: backward on (v, do, q), the state's gradient transposed
    AttnPass &y = a.p[1];
    y.q = p->v, y.k = d_o, y.v = p->q, y.o = g > 1 ? w.part[0] : dk;
    strides_of(y.qs, p->v_strides);
    strides_of(y.ks, d_o_strides);
    strides_of(y.vs, p->q_strides);
    dense_strides(y.os, p->T, p->H, p->Dk);
    y.qg = g, y.kg = y.vg = 1;
    y.dq = dV, y.dv = dK;
    y.s_in = dstate_out, y.s_row = 1, y.s_col = dV;
    y.p_scale = y.w_scale = p->scale, y.i_scale = 1.0f;
    y.shift = 1, y.rev = 1, y.o_f32 = g > 1;
    y.seg = w.seg[1];
    // dv: backward on (k, q, do); its final state is the gradient of the initial one
    AttnPass &z = a.p[2];
    z.q = p->k, z.k = p->q, z.v = d_o, z.o = g > 1 ? w.part[1] : dv;
    strides_of(z.qs, p->k_strides);
    strides_of(z.ks, p->q_strides);
    strides_of(z.vs, d_o_strides);
    dense_strides(z.os, p->T, p->H, p->Dv);
    z.qg = g, z.kg = z.vg = 1;
    z.dq = dK, z.dv = dV;
    z.s_in = dstate_out, z.s_out = dstate, z.s_row = dV, z.s_col = 1;
    z.p_scale = z.w_scale = p->scale, z.i_scale = 1.0f;
    z.shift = 1, z.rev = 1, z.o_f32 = g > 1;
    z.seg = w.seg[2];
    if (!run_passes(a, 3, p->dtype, s)) return at_fail(LIFB_ERR_CUDA, what, "launch failed");
    if (g > 1) {
        const int64_t rows = p->B * p->T * p->Hk;
        auto blocks = [&](int64_t d) { return (unsigned)std::min<int64_t>((rows * d + 255) / 256, kAtSms * 16); };
        count_launches(2);
        if (p->dtype == LIFB_F32) {
            k_attn_group<<<blocks(dK), 256, 0, s>>>(w.part[0], (float *)dk, rows, g, dK);
            k_attn_group<<<blocks(dV), 256, 0, s>>>(w.part[1], (float *)dv, rows, g, dV);
        } else {
            k_attn_group<<<blocks(dK), 256, 0, s>>>(w.part[0], (__nv_bfloat16 *)dk, rows, g, dK);
            k_attn_group<<<blocks(dV), 256, 0, s>>>(w.part[1], (__nv_bfloat16 *)dv, rows, g, dV);
        }
    }
    if (cudaGetLastError() != cudaSuccess) return at_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}

namespace lifb {
namespace {

template <typename T>
void step_launch(const lifb_leaky_attn_step_args &p, void *o, float *state, cudaStream_t s)
{
    const bool wide = p.Dv % 4 == 0 && p.state_strides[0] % 4 == 0 && p.state_strides[1] % 4 == 0 && aligned16(state) &&
                      p.v_strides[0] % 4 == 0 && p.v_strides[1] % 4 == 0 && (uintptr_t)p.v % (4 * sizeof(T)) == 0 &&
                      (uintptr_t)o % (4 * sizeof(T)) == 0;
    const int vec = wide ? 4 : 1, cols = (int)(p.Dv + vec - 1) / vec;
    const int cv = std::min(cols, 16), threads = kAtThreads / cv * cv;
    const dim3 grid((unsigned)(p.B * p.H), (unsigned)((cols + cv - 1) / cv));
    auto kern = wide ? k_attn_step<T, 4> : k_attn_step<T, 1>;
    count_launches(1);
    kern<<<grid, threads, 0, s>>>((const T *)p.q, (const T *)p.k, (const T *)p.v, (T *)o, p.log_decay, state, p.slots,
                                  p.n_slots, (int)p.H, (int)(p.H / p.Hk), (int)p.Dk, (int)p.Dv, cv, p.q_strides[0],
                                  p.q_strides[1], p.k_strides[0], p.k_strides[1], p.v_strides[0], p.v_strides[1],
                                  p.state_strides[0], p.state_strides[1], p.scale);
}

}  // namespace
}  // namespace lifb

extern "C" int lifb_leaky_attn_step(const lifb_leaky_attn_step_args *p, void *o, float *state, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_leaky_attn_step");
    const char *what = "lifb_leaky_attn_step";
    if (!p) return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null arguments");
    if (p->B < 0 || p->H < 0 || p->Hk < 0 || p->Dk < 0 || p->Dv < 0 || p->n_slots < 0)
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "negative shape");
    if (!dtype_bytes(p->dtype)) return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "unknown dtype");
    if (p->H > 0 && (p->Hk <= 0 || p->H % p->Hk))
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "H must be a multiple of Hk");
    if (p->Dk > kAttnMaxDim || p->Dv > kAttnMaxDim)
        return at_fail(LIFB_ERR_UNSUPPORTED, what, "head widths up to 128");
    if (p->B * p->H >= (int64_t(1) << 31)) return at_fail(LIFB_ERR_UNSUPPORTED, what, "needs B * H < 2^31");
    if (!p->slots && p->n_slots < p->B)
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "without slots the cache holds one state for each sequence");
    if (p->B == 0 || p->H == 0 || p->Dv == 0) return LIFB_OK;
    if (!p->q || !p->k || !p->v || !p->log_decay || !o || !state)
        return at_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    LIFB_BY_DTYPE(p->dtype, T, step_launch<T>(*p, o, state, (cudaStream_t)stream));
    if (cudaGetLastError() != cudaSuccess) return at_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}
