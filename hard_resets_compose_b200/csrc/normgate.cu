// The norms around a block, its gate and its scaled residual, in one pass:
//
//   y  = rmsnorm(h) * post        rmsnorm(z) = z * r(z), r(z) = 1/sqrt(mean z^2 + eps)
//   x' = x + s * a * y            a = 1, or act(gate): elementwise or one value for a row
//   n  = rmsnorm(x') * pre        the next block's input
//
// and its backward from (dx', dn):
//
//   t    = dx' + r(x') * (u - xh * mean(u * xh))    u = dn * pre, xh = x' r(x')
//   dx   = t,   dgate = s * t * y * act'(gate)  (summed over the row if it is one value)
//   dh   = r(h) * (w - hh * mean(w * hh))           w = s * a * t * post, hh = h r(h)
//   dpre = sum over rows of dn * xh,   dpost = sum over rows of s * a * t * hh
//
// Everything is bound by memory: the forward reads x, h, gate and writes x', n;
// the backward reads dx', dn, x, h, gate and writes dx, dh, dgate.  A row stays
// in registers between its two means, so each tensor crosses memory once; the
// backward forms x' again from x, h and gate in fp32 rather than read the
// rounded x' (the same bytes, and dpre keeps fp32 accuracy).  The forward keeps
// r(h) and r(x') of each row, 8 bytes.  A group of TPR threads (a power of two)
// owns a row, NIT vectors of VEC elements a thread; groups walk the rows with
// a grid stride, so that the weights stay in registers and the backward adds
// its rows' parts of dpre and dpost there, in row order; the groups' and then the
// blocks' sums (fp32; a second launch) are added in a fixed order.
// Measured: bf16 [32768, 2048] with an elementwise gate 109 us forward (104 us at the
// copy rate) and 224 us backward (166): the backward's 65 instructions an element leave
// the memory waiting a quarter of the time; fp32 [65536, 256] with a row's gate 50 us
// (42) and 75 us (62).
#include <algorithm>
#include <initializer_list>

#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "f32x2.cuh"
#include "seq_types.cuh"
#include "tma.cuh"

namespace lifb {

namespace {

constexpr int kNgThreads = 256;      // of a block, where a row needs no more
constexpr int kNgMaxThreads = 512;   // of a block of a longer row: 128 registers a thread
constexpr int kNgMaxElems = 16;      // of a row in one thread
constexpr int kNgSms = 148;
constexpr int kNgReduceRows = 16;    // groups of partial sums added by one block of the second launch

enum Act : int { kActSilu = 0, kActSigmoid = 1, kActLinear = 2 };

struct NormArgs {
    const void *x, *h, *gate;
    const void *post, *pre;
    int64_t sx, sh, sg, sdx, sdn;  // row strides, in elements
    void *xo, *n;                  // [R, D] contiguous
    float *rstd;                   // [2][R]: r(h), r(x')
    const void *dxo, *dn;
    void *dx, *dh, *dgate;
    float *part;  // [blocks][2][D]
    int64_t R, D;
    float scale, eps;
    int act, gate_row, w_f32;
};

// Blocks of a kernel that an SM holds; registers are spread accordingly.
// (Single elements take twice the registers of packed ones.)
__host__ __device__ constexpr int norm_blocks_per_sm(bool bwd, int threads, int vec, int nit)
{
    const int elems = vec == 1 ? 2 * nit : vec * nit;
    return threads > kNgThreads || elems > 16 ? 1 : elems > 8 ? 2 : elems > 4 ? (bwd ? 2 : 3) : (bwd ? 4 : 5);
}

}  // namespace

// Sums NV values over the tpr threads of a row (a power of two); every thread gets
// them.  `sh`: 2 * NV * 32 floats, halves used alternately by `flip`.
template <int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], int tpr, float *sh, int &flip)
{
    if (tpr >= 32) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < NV; i++) v[i] += __shfl_xor_sync(~0u, v[i], o);
        }
    } else {
        for (int o = tpr >> 1; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < NV; i++) v[i] += __shfl_xor_sync(~0u, v[i], o);
        }
    }
    if (tpr > 32) {
        // rows of one block reduce in lockstep: every group makes the same calls
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wpr = tpr >> 5;
        float *buf = sh + flip * NV * 32;
        flip ^= 1;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) buf[i * 32 + warp] = v[i];
        }
        __syncthreads();
        const int at = (warp & -wpr) + (lane & (wpr - 1));
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] = buf[i * 32 + at];
        for (int o = wpr >> 1; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < NV; i++) v[i] += __shfl_xor_sync(~0u, v[i], o);
        }
    }
}

// exp(-g).  fp32 rows: expf.  Rows of 16 bits: the 2-ulp power of two; rounding its exponent
// puts |g| 2^-24 into the result, 2^-17 at |g| = 128, where a bf16 or fp16 output is rounded
// by 2^-9 or 2^-12 (with expf and the division their norms waited for them instead of memory).
template <typename T>
__device__ __forceinline__ float exp_minus(float g)
{
    return sizeof(T) == 4 ? expf(-g) : ex2_approx(-1.4426950408889634f * g);
}

// sigmoid(g), with the 1-ulp reciprocal
template <typename T>
__device__ __forceinline__ float sigmoid(float g) { return rcp_approx(1.0f + exp_minus<T>(g)); }

// act(g) and act'(g) of one value, a row's gate
template <typename T>
__device__ __forceinline__ float act_value(int act, float g)
{
    return act == kActLinear ? g : act == kActSilu ? g * sigmoid<T>(g) : sigmoid<T>(g);
}
template <typename T>
__device__ __forceinline__ float act_grad(int act, float g)
{
    const float sg = sigmoid<T>(g);
    return act == kActLinear ? 1.0f : act == kActSilu ? sg + g * (sg - sg * sg) : sg - sg * sg;
}

// The same of a pair (in packed arithmetic): act(g), and with `da` act'(g).
template <typename T>
__device__ __forceinline__ uint64_t act_pair(int act, uint64_t g, uint64_t *da)
{
    if (act == kActLinear) {
        if (da) *da = two(1.0f, 1.0f);
        return g;
    }
    float z0, z1;
    if (sizeof(T) == 4) {
        both(g, z0, z1);
        z0 = expf(-z0);
        z1 = expf(-z1);
    } else {
        both(mul2(g, two(-1.4426950408889634f, -1.4426950408889634f)), z0, z1);
        z0 = ex2_approx(z0);
        z1 = ex2_approx(z1);
    }
    both(add2(two(z0, z1), two(1.0f, 1.0f)), z0, z1);
    const uint64_t sg = two(rcp_approx(z0), rcp_approx(z1));
    if (da) {
        const uint64_t d = fma2(mul2(sg, two(-1.0f, -1.0f)), sg, sg);  // sg - sg^2
        *da = act == kActSilu ? fma2(g, d, sg) : d;
    }
    return act == kActSilu ? mul2(g, sg) : sg;
}

// A row's elements of one thread, NIT vectors of VEC, as pairs in that order.
template <typename T, int VEC, int NIT>
struct Row {
    static constexpr int kPairs = VEC * NIT / 2;
    uint64_t v[kPairs];
};

// A row's vectors of one tensor, as they are in memory: loaded for the next row
// while the present one waits for its sums.  Absent tensors and columns are zero and
// never loaded; a row past the last is loaded as the last one and then cleared.
template <typename T, int VEC, int NIT>
struct RowPart {
    Pack<T, VEC> p[NIT];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < NIT; i++) p[i].zero();
    }
    __device__ __forceinline__ void load(const void *row, int step, const bool (&in)[NIT])
    {
#pragma unroll
        for (int i = 0; i < NIT; i++)
            if (in[i]) p[i].load((const T *)row + i * step);
    }
    __device__ __forceinline__ void get(Row<T, VEC, NIT> &x) const
    {
        float f[NIT][VEC];
#pragma unroll
        for (int i = 0; i < NIT; i++) p[i].get(f[i]);
#pragma unroll
        for (int i = 0; i < VEC * NIT; i += 2) x.v[i / 2] = two(f[i / VEC][i % VEC], f[(i + 1) / VEC][(i + 1) % VEC]);
    }
};

template <typename T, int VEC, int NIT>
__device__ __forceinline__ void store_row(const Row<T, VEC, NIT> &x, void *base, int64_t at, int step,
                                          const bool (&in)[NIT])
{
    T *row = (T *)base + at;
    float f[NIT][VEC];
#pragma unroll
    for (int i = 0; i < VEC * NIT; i += 2) both(x.v[i / 2], f[i / VEC][i % VEC], f[(i + 1) / VEC][(i + 1) % VEC]);
#pragma unroll
    for (int i = 0; i < NIT; i++)
        if (in[i]) store_f32(row + i * step, f[i]);
}

// A weight's elements of this thread, zero past the row's end.
template <typename T, int VEC, int NIT>
__device__ __forceinline__ void load_weight(Row<T, VEC, NIT> &x, const void *w, int f32, int c0, int step, int D)
{
    float f[NIT][VEC];
#pragma unroll
    for (int i = 0; i < NIT; i++)
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const int c = c0 + i * step;
            f[i][e] = c >= D || !w ? 0.0f : f32 ? ((const float *)w)[c + e] : to_f32(((const T *)w)[c + e]);
        }
#pragma unroll
    for (int i = 0; i < VEC * NIT; i += 2) x.v[i / 2] = two(f[i / VEC][i % VEC], f[(i + 1) / VEC][(i + 1) % VEC]);
}

// GATE: the gate's form at compile time (0 none, 1 elementwise, 2 one value a row) or -1
// (as the arguments say); ACT: its activation, or -1.
template <typename T, int VEC, int NIT, int MAXT, int GATE, int ACT>
__global__ void __launch_bounds__(MAXT, norm_blocks_per_sm(false, MAXT, VEC, NIT))
    k_norm_fwd(const __grid_constant__ NormArgs a, int tpr)
{
    using R = Row<T, VEC, NIT>;
    constexpr int P = R::kPairs;
    __shared__ float sh[2 * 32];
    int flip = 0;
    const int lane = threadIdx.x & (tpr - 1), c0 = lane * VEC, step = tpr * VEC, D = (int)a.D;
    const int64_t groups = blockDim.x / tpr, g = threadIdx.x / tpr, stride = gridDim.x * groups;
    const bool full_gate = GATE == 1 || (GATE < 0 && a.gate && !a.gate_row);
    const bool row_gate = GATE == 2 || (GATE < 0 && a.gate && a.gate_row);
    const int act = ACT >= 0 ? ACT : a.act;
    const float inv_d = 1.0f / (float)a.D;
    R post, pre;
    load_weight(post, a.h ? a.post : nullptr, a.w_f32, c0, step, D);
    load_weight(pre, a.n ? a.pre : nullptr, a.w_f32, c0, step, D);
    bool in[NIT];
#pragma unroll
    for (int i = 0; i < NIT; i++) in[i] = c0 + i * step < D;
    RowPart<T, VEC, NIT> nx, nh, ng;
    nx.clear();
    nh.clear();
    ng.clear();
    float grow = 0.0f;
    auto fetch = [&](int64_t r) {
        r = min(r, a.R - 1);
        nx.load((const T *)a.x + r * a.sx + c0, step, in);
        if (a.h) nh.load((const T *)a.h + r * a.sh + c0, step, in);
        if (full_gate) ng.load((const T *)a.gate + r * a.sg + c0, step, in);
        if (row_gate) grow = to_f32(((const T *)a.gate)[r * a.sg]);
    };
    fetch(blockIdx.x * groups + g);
    // every group of a block makes the same number of rounds
    for (int64_t r0 = blockIdx.x * groups; r0 < a.R; r0 += stride) {
        const int64_t r = r0 + g;
        const bool on = r < a.R;
        R x, h, gt;
        nx.get(x);
        nh.get(h);
        if (full_gate) ng.get(gt);
        const float arow = row_gate ? act_value<T>(a.act, grow) : 1.0f;
        fetch(r + stride);
        if (a.h) {
            uint64_t s2 = 0;
#pragma unroll
            for (int i = 0; i < P; i++) s2 = fma2(h.v[i], h.v[i], s2);
            float ss[1] = {sum_of(s2)};
            row_sum(ss, tpr, sh, flip);
            const float rh = rsqrtf(ss[0] * inv_d + a.eps);
            if (on && lane == 0 && a.rstd) a.rstd[r] = rh;
            const float k = a.scale * rh * arow;
            const uint64_t kk = two(k, k);
#pragma unroll
            for (int i = 0; i < P; i++) {
                uint64_t y = mul2(h.v[i], post.v[i]);
                if (full_gate) y = mul2(y, act_pair<T>(act, gt.v[i], nullptr));
                x.v[i] = fma2(kk, y, x.v[i]);
            }
            if (on) store_row(x, a.xo, r * a.D + c0, step, in);
        }
        if (a.n) {
            uint64_t s2 = 0;
#pragma unroll
            for (int i = 0; i < P; i++) s2 = fma2(x.v[i], x.v[i], s2);
            float ss[1] = {sum_of(s2)};
            row_sum(ss, tpr, sh, flip);
            const float rx = rsqrtf(ss[0] * inv_d + a.eps);
            if (on && lane == 0 && a.rstd) a.rstd[a.R + r] = rx;
            const uint64_t k = two(rx, rx);
#pragma unroll
            for (int i = 0; i < P; i++) x.v[i] = mul2(mul2(x.v[i], k), pre.v[i]);
            if (on) store_row(x, a.n, r * a.D + c0, step, in);
        }
    }
}

// The weights and the sums of their gradients lie in shared memory in vectors of four
// elements, vector q of a row's thread `lane` at (q * tpr + lane) * 4: registers are
// what limits the rows in flight.
template <typename T, int VEC, int NIT, int MAXT, int GATE, int ACT>
__global__ void __launch_bounds__(MAXT, norm_blocks_per_sm(true, MAXT, VEC, NIT))
    k_norm_bwd(const __grid_constant__ NormArgs a, int tpr)
{
    using R = Row<T, VEC, NIT>;
    constexpr int P = R::kPairs, Q = P / 2;
    constexpr bool kAhead = VEC * NIT <= 8;  // the next row's loads before this one's sums
    __shared__ float sh[2 * 2 * 32];
    extern __shared__ float4 ng_smem[];
    int flip = 0;
    const int lane = threadIdx.x & (tpr - 1), c0 = lane * VEC, step = tpr * VEC, D = (int)a.D;
    const int groups = blockDim.x / tpr, g = threadIdx.x / tpr;
    const int64_t stride = (int64_t)gridDim.x * groups;
    const bool full_gate = GATE == 1 || (GATE < 0 && a.gate && !a.gate_row);
    const bool row_gate = GATE == 2 || (GATE < 0 && a.gate && a.gate_row);
    const int act = ACT >= 0 ? ACT : a.act;
    const float inv_d = 1.0f / (float)a.D;
    float4 *post = ng_smem + lane, *pre = post + Q * tpr, *dpost = pre + (1 + 2 * g) * Q * tpr, *dpre = dpost + Q * tpr;
    if (g == 0) {
        R w;
        load_weight(w, a.h ? a.post : nullptr, a.w_f32, c0, step, D);
        for (int q = 0; q < Q; q++) reinterpret_cast<ulonglong2 *>(post)[q * tpr] = make_ulonglong2(w.v[2 * q], w.v[2 * q + 1]);
        load_weight(w, a.dn ? a.pre : nullptr, a.w_f32, c0, step, D);
        for (int q = 0; q < Q; q++) reinterpret_cast<ulonglong2 *>(pre)[q * tpr] = make_ulonglong2(w.v[2 * q], w.v[2 * q + 1]);
    }
    for (int q = 0; q < Q; q++) dpost[q * tpr] = dpre[q * tpr] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    auto four = [&](const float4 *p, int q) { return *reinterpret_cast<const ulonglong2 *>(p + q * tpr); };
    auto add_four = [&](float4 *p, int q, uint64_t a0, uint64_t b0, uint64_t a1, uint64_t b1) {
        ulonglong2 *at = reinterpret_cast<ulonglong2 *>(p + q * tpr);
        const ulonglong2 z = *at;
        *at = make_ulonglong2(fma2(a0, b0, z.x), fma2(a1, b1, z.y));
    };
    bool in[NIT];
#pragma unroll
    for (int i = 0; i < NIT; i++) in[i] = c0 + i * step < D;
    RowPart<T, VEC, NIT> nt, nu, nx, nh, ng;
    nt.clear();
    nu.clear();
    nx.clear();
    nh.clear();
    ng.clear();
    float nrh = 0.0f, nrx = 0.0f, ngr = 0.0f;
    auto fetch = [&](int64_t row) {
        const int64_t r = min(row, a.R - 1);
        if (!kAhead) {  // nothing of a row lives past it
            nt.clear();
            nu.clear();
            nx.clear();
            nh.clear();
            ng.clear();
        }
        if (a.dn) {
            nu.load((const T *)a.dn + r * a.sdn + c0, step, in);
            nx.load((const T *)a.x + r * a.sx + c0, step, in);
            nrx = a.rstd[a.R + r];
        }
        if (a.h) {
            nh.load((const T *)a.h + r * a.sh + c0, step, in);
            nrh = a.rstd[r];
        }
        if (full_gate) ng.load((const T *)a.gate + r * a.sg + c0, step, in);
        if (a.dxo) nt.load((const T *)a.dxo + r * a.sdx + c0, step, in);
        if (row_gate) ngr = to_f32(((const T *)a.gate)[r * a.sg]);
        if (row >= a.R) {  // adds nothing to the sums
            nt.clear();
            nu.clear();
            nx.clear();
            nh.clear();
        }
    };
    if (kAhead) fetch(blockIdx.x * groups + g);
    for (int64_t r0 = blockIdx.x * groups; r0 < a.R; r0 += stride) {
        const int64_t r = r0 + g;
        const bool on = r < a.R;
        if (!kAhead) fetch(r);
        // t: dx', then the gradient of x'; hh: h r(h); av, da: the gate's act and act'
        R t, hh, av, da, x, u;
        const float rh = nrh, rx = nrx, grow = ngr;
        nt.get(t);
        nu.get(u);
        nx.get(x);
        nh.get(hh);
        if (full_gate) ng.get(av);
        if (kAhead) fetch(r + stride);
        const float arow = row_gate ? act_value<T>(a.act, grow) : 1.0f;
        if (a.h) {
            const uint64_t k = two(rh, rh);
#pragma unroll
            for (int i = 0; i < P; i++) {
                hh.v[i] = mul2(hh.v[i], k);
                if (full_gate) av.v[i] = act_pair<T>(act, av.v[i], &da.v[i]);
            }
        }
        if (a.dn) {
            const float kf = a.scale * arow;
            const uint64_t k = two(kf, kf), kx = two(rx, rx);
            uint64_t m2 = 0;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                const ulonglong2 wp = four(pre, q);
                ulonglong2 ws = make_ulonglong2(0, 0);
                if (a.h) ws = four(post, q);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int i = 2 * q + j;
                    if (a.h) {
                        uint64_t y = mul2(hh.v[i], j ? ws.y : ws.x);
                        if (full_gate) y = mul2(y, av.v[i]);
                        x.v[i] = fma2(k, y, x.v[i]);
                    }
                    x.v[i] = mul2(x.v[i], kx);
                }
                add_four(dpre, q, u.v[2 * q], x.v[2 * q], u.v[2 * q + 1], x.v[2 * q + 1]);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int i = 2 * q + j;
                    u.v[i] = mul2(u.v[i], j ? wp.y : wp.x);
                    m2 = fma2(u.v[i], x.v[i], m2);
                }
            }
            float m[1] = {sum_of(m2)};
            row_sum(m, tpr, sh, flip);
            const float mu = -m[0] * inv_d;
            const uint64_t mm = two(mu, mu);
#pragma unroll
            for (int i = 0; i < P; i++) t.v[i] = fma2(kx, fma2(x.v[i], mm, u.v[i]), t.v[i]);
        }
        if (on && a.dx) store_row(t, a.dx, r * a.D + c0, step, in);
        if (a.h) {
            const uint64_t k = two(a.scale, a.scale), ka = two(arow, arow);
            uint64_t m2 = 0, row2 = 0;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                const ulonglong2 w = four(post, q);
                uint64_t ai[2], sh_[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int i = 2 * q + j;
                    const uint64_t wj = j ? w.y : w.x, st = mul2(t.v[i], k);
                    sh_[j] = mul2(st, hh.v[i]);
                    const uint64_t ty = mul2(sh_[j], wj);
                    ai[j] = full_gate ? av.v[i] : ka;
                    if (full_gate) da.v[i] = mul2(ty, da.v[i]);
                    if (row_gate) row2 = add2(row2, ty);
                    t.v[i] = mul2(mul2(st, ai[j]), wj);
                    m2 = fma2(t.v[i], hh.v[i], m2);
                }
                add_four(dpost, q, ai[0], sh_[0], ai[1], sh_[1]);
            }
            if (on && full_gate && a.dgate) store_row(da, a.dgate, r * a.D + c0, step, in);
            float m[2] = {sum_of(m2), row_gate ? sum_of(row2) : 0.0f};
            row_sum(m, tpr, sh, flip);
            const float mw = -m[0] * inv_d;
            const uint64_t mm = two(mw, mw), kh = two(rh, rh);
#pragma unroll
            for (int i = 0; i < P; i++) t.v[i] = mul2(kh, fma2(hh.v[i], mm, t.v[i]));
            if (on && a.dh) store_row(t, a.dh, r * a.D + c0, step, in);
            if (row_gate && a.dgate && on && lane == 0) ((T *)a.dgate)[r] = from_f32<T>(m[1] * act_grad<T>(a.act, grow));
        }
    }
    if (!a.part) return;
    // the block's sums: its groups' parts added in order, dpost then dpre
    __syncthreads();
    float *part = a.part + (int64_t)blockIdx.x * 2 * D;
    const float *sums = reinterpret_cast<const float *>(ng_smem + 2 * Q * tpr);  // [groups][2][Q][tpr][4]
    for (int j = threadIdx.x; j < 2 * 4 * Q * tpr; j += blockDim.x) {
        const int which = j / (4 * Q * tpr), k = j - which * (4 * Q * tpr);
        const int f = k / (4 * tpr) * 4 + k % 4, l = k / 4 % tpr;  // the element of thread l
        const int c = l * VEC + f / VEC * step + f % VEC;
        if (c >= D) continue;
        float v = 0.0f;
        for (int i = 0; i < groups; i++) v += sums[(int64_t)i * 8 * Q * tpr + j];
        part[which * D + c] = v;
    }
}

// Adds the blocks' parts column by column, in order: 32 columns a block, one
// warp for every kNgReduceRows-th part, then the warps' sums.
template <typename T>
__global__ void __launch_bounds__(32 * kNgReduceRows)
    k_norm_weight_grads(const float *__restrict__ part, int64_t parts, int64_t D, void *dpost, void *dpre, int w_f32)
{
    __shared__ float s[kNgReduceRows][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // of 2 D: dpost, then dpre
    float v = 0.0f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int64_t p = warp; p < parts; p += kNgReduceRows) v += part[p * 2 * D + c];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < 2 * D) {
        v = 0.0f;
        for (int w = 0; w < kNgReduceRows; w++) v += s[w][lane];
        void *out = c < D ? dpost : dpre;
        const int64_t at = c < D ? c : c - D;
        if (out) {
            if (w_f32) ((float *)out)[at] = v;
            else ((T *)out)[at] = from_f32<T>(v);
        }
    }
}

namespace {

// How a row is spread: VEC, NIT and the threads of a row; false if it is too long.
struct NormShape {
    int vec, nit, tpr, threads;
};

// A row takes as few threads as hold it at 16 (fp32 forward: 8) elements each,
// in one warp if it can: a row costs each thread some 150 instructions besides its
// elements (bf16 rows of 2048: forward 150 us with 8 elements a thread, 109 us with 16).
// Rows that are read element by element take more threads instead, and so do long rows
// of 8-byte fp32 vectors, whose forward would spill at 16 (8000 rows of 3002: 165 us in
// 256 threads, 85 in 512; 16-byte vectors: 66 against 82).  Narrower vectors where 16
// bytes do not fit: bf16 [30000, 1028] with an elementwise gate, by single elements 220
// us forward and 474 backward, by 8 bytes 123 and 229, by 4 ([30000, 1030]) 184 and 290.
bool norm_shape(int64_t D, int vec, int elem, bool bwd, NormShape &s)
{
    s.vec = vec;
    const int widest = 16 / elem;
    const bool wide = vec > 1;
    const int64_t vecs = (D + s.vec - 1) / s.vec;
    // the row over `tpr` threads of a block of `threads`, with as few elements each as hold it
    auto spread = [&](int threads, int tpr, int elems) {
        s.threads = threads;
        s.tpr = tpr;
        // 16-byte vectors: any number of them; single elements: 4, 8 or 16; between: 8 or 16 elements
        s.nit = vec == widest ? 1 : wide ? 8 / vec : 4;
        while (s.nit * s.vec < elems && (int64_t)s.tpr * s.nit < vecs) s.nit *= 2;
        return (int64_t)s.tpr * s.nit >= vecs;
    };
    // elements a thread at most before the row takes more threads
    auto most = [&](int tpr) {
        if (tpr < 32) return wide && vec < widest ? 8 : vec;  // part of a warp: the fewest there are
        if (!wide) return tpr == 32 ? kNgMaxElems : tpr < kNgThreads ? 4 : 8;
        return elem == 2 || bwd ? kNgMaxElems : 8;
    };
    for (int tpr = 8; tpr <= kNgThreads; tpr *= 2)
        if (spread(kNgThreads, tpr, most(tpr))) return true;
    if ((!wide || (elem == 4 && vec == 2)) && spread(kNgMaxThreads, kNgMaxThreads, 8)) return true;
    return spread(kNgThreads, kNgThreads, kNgMaxElems) || spread(kNgMaxThreads, kNgMaxThreads, kNgMaxElems);
}

int64_t norm_blocks(const NormShape &s, int64_t R, bool bwd)
{
    const int64_t groups = s.threads / s.tpr;
    const int64_t per_sm = norm_blocks_per_sm(bwd, s.threads, s.vec, s.nit);
    return std::max<int64_t>(1, std::min<int64_t>((R + groups - 1) / groups, kNgSms * per_sm));
}

template <typename T, int VEC, int NIT, int MAXT, int GATE, int ACT = -1>
bool norm_launch(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    const unsigned blocks = (unsigned)norm_blocks(sh, a.R, bwd);
    if (bwd) {
        // weights, and each group's sums: 2 * (1 + groups) rows of tpr * VEC * NIT floats
        const size_t smem = (size_t)2 * (1 + sh.threads / sh.tpr) * sh.tpr * VEC * NIT * 4;
        // the kernel's limit is the most that any row takes (tpr = MAXT; 128 KB at most): the
        // limit is one for all threads, and a call's own size could lower it under another's launch
        auto kern = k_norm_bwd<T, VEC, NIT, MAXT, GATE, ACT>;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 2 * MAXT * VEC * NIT * 4) !=
            cudaSuccess)
            return false;
        count_launches(1);
        kern<<<blocks, MAXT, smem, s>>>(a, sh.tpr);
    } else {
        count_launches(1);
        k_norm_fwd<T, VEC, NIT, MAXT, GATE, ACT><<<blocks, MAXT, 0, s>>>(a, sh.tpr);
    }
    return true;
}

template <typename T, int VEC, int NIT>
bool norm_gate(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    if (sh.threads == kNgMaxThreads) {
        if constexpr (VEC * NIT == kNgMaxElems || (VEC * NIT == 8 && (VEC == 1 || (VEC == 2 && sizeof(T) == 4))))
            return norm_launch<T, VEC, NIT, kNgMaxThreads, -1>(bwd, a, sh, s);
        else
            return false;  // norm_shape gives no such row
    } else if constexpr (VEC * sizeof(T) != 16) {
        return norm_launch<T, VEC, NIT, kNgThreads, -1>(bwd, a, sh, s);
    } else if (!a.gate) {
        return norm_launch<T, VEC, NIT, kNgThreads, 0>(bwd, a, sh, s);
    } else if (a.gate_row) {
        return norm_launch<T, VEC, NIT, kNgThreads, 2>(bwd, a, sh, s);
    } else if (a.act == kActSilu) {
        return norm_launch<T, VEC, NIT, kNgThreads, 1, kActSilu>(bwd, a, sh, s);
    } else if (a.act == kActSigmoid) {
        return norm_launch<T, VEC, NIT, kNgThreads, 1, kActSigmoid>(bwd, a, sh, s);
    } else {
        return norm_launch<T, VEC, NIT, kNgThreads, 1, kActLinear>(bwd, a, sh, s);
    }
}

template <typename T>
bool norm_run(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    if (sh.vec == 1) {
        if (sh.nit == 4) return norm_gate<T, 1, 4>(bwd, a, sh, s);
        else if (sh.nit == 8) return norm_gate<T, 1, 8>(bwd, a, sh, s);
        else return norm_gate<T, 1, 16>(bwd, a, sh, s);
    } else if (sh.vec == 2) {
        if (sh.nit == 4) return norm_gate<T, 2, 4>(bwd, a, sh, s);
        else return norm_gate<T, 2, 8>(bwd, a, sh, s);
    } else if (sh.vec < VEC) {
        if constexpr (VEC == 8) {
            if (sh.nit == 2) return norm_gate<T, 4, 2>(bwd, a, sh, s);
            else return norm_gate<T, 4, 4>(bwd, a, sh, s);
        }
    } else if (sh.nit == 1) {
        return norm_gate<T, VEC, 1>(bwd, a, sh, s);
    } else if (sh.nit == 2) {
        return norm_gate<T, VEC, 2>(bwd, a, sh, s);
    } else if constexpr (VEC == 4) {
        return norm_gate<T, VEC, 4>(bwd, a, sh, s);
    }
    return false;
}

// Elements of a vector that D, the strides and the addresses (null: absent) allow.
int norm_vec(int elem, int64_t D, std::initializer_list<int64_t> strides, std::initializer_list<const void *> ptrs)
{
    int vec = 16 / elem;
    for (; vec > 1; vec /= 2) {
        bool ok = D % vec == 0;
        for (int64_t st : strides) ok = ok && st % vec == 0;
        for (const void *p : ptrs) ok = ok && (uintptr_t)p % (vec * elem) == 0;
        if (ok) break;
    }
    return vec;
}

int norm_fail(int status, const char *what, const char *why)
{
    char msg[160];
    snprintf(msg, sizeof msg, "%s: %s", what, why);
    set_last_error(msg);
    return status;
}

int norm_check(const char *what, const lifb_norm_gate *p, NormArgs &a)
{
    if (!p) return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null arguments");
    if (p->R < 0 || p->D < 0) return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "negative shape");
    if (!dtype_bytes(p->dtype) || (p->weight_dtype != LIFB_F32 && p->weight_dtype != p->dtype))
        return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "weights are fp32 or of the rows' type");
    if (p->act < kActSilu || p->act > kActLinear) return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "unknown act");
    if (p->gate_cols != 0 && p->gate_cols != 1 && p->gate_cols != p->D)
        return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "the gate has D columns, one, or none");
    a = {};
    a.x = p->x;
    a.h = p->h;
    a.gate = p->gate_cols ? p->gate : nullptr;
    a.post = p->post;
    a.pre = p->pre;
    a.sx = p->x_stride;
    a.sh = p->h_stride;
    a.sg = p->gate_stride;
    a.rstd = p->rstd;
    a.R = p->R;
    a.D = p->D;
    a.scale = p->scale;
    a.eps = p->eps;
    a.act = p->act;
    a.gate_row = p->gate_cols == 1 && p->D != 1;
    a.w_f32 = p->weight_dtype == LIFB_F32;
    return LIFB_OK;
}

}  // namespace

}  // namespace lifb

extern "C" int lifb_norm_gate_fwd(const lifb_norm_gate *p, void *xo, void *n, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_norm_gate_fwd");
    const char *what = "lifb_norm_gate_fwd";
    NormArgs a;
    if (int st = norm_check(what, p, a)) return st;
    if (a.R == 0 || a.D == 0) return LIFB_OK;
    a.xo = xo;
    a.n = n;
    if (!a.x || (a.h && (!a.post || !xo)) || (n && !a.pre) || (p->gate_cols && !p->gate) || (!a.h && !n))
        return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    const bool gate = a.gate && !a.gate_row;
    const int elem = (int)dtype_bytes(p->dtype);
    const int vec = norm_vec(elem, a.D, {a.sx, a.h ? a.sh : 0, gate ? a.sg : 0}, {a.x, xo, n, a.h, gate ? a.gate : nullptr});
    NormShape sh;
    if (!norm_shape(a.D, vec, elem, false, sh))
        return norm_fail(LIFB_ERR_UNSUPPORTED, what, "rows longer than 8192 elements");
    bool ok = false;
    LIFB_BY_DTYPE(p->dtype, T, ok = norm_run<T>(false, a, sh, (cudaStream_t)stream));
    if (cudaGetLastError() != cudaSuccess || !ok) return norm_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}

extern "C" size_t lifb_norm_gate_bwd_workspace_bytes(int64_t R, int64_t D, int dtype)
{
    using namespace lifb;
    if (R <= 0 || D <= 0 || !dtype_bytes(dtype)) return 0;
    size_t most = 0;  // of any vectors
    for (int vec = 16 / (int)dtype_bytes(dtype); vec > 0; vec /= 2) {
        NormShape sh;
        if (norm_shape(D, vec, (int)dtype_bytes(dtype), true, sh))
            most = std::max(most, (size_t)norm_blocks(sh, R, true) * 2 * D * 4);
    }
    return most;
}

extern "C" int lifb_norm_gate_bwd(const lifb_norm_gate *p, const void *dxo, int64_t dxo_stride, const void *dn,
                                  int64_t dn_stride, void *dx, void *dh, void *dgate, void *dpost, void *dpre,
                                  void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_norm_gate_bwd");
    const char *what = "lifb_norm_gate_bwd";
    NormArgs a;
    if (int st = norm_check(what, p, a)) return st;
    cudaStream_t s = (cudaStream_t)stream;
    const bool weights = dpost || dpre;
    if (a.D == 0) return LIFB_OK;
    if (a.R == 0) {
        const size_t nb = (size_t)a.D * (a.w_f32 ? 4 : dtype_bytes(p->dtype));
        if ((dpost && cudaMemsetAsync(dpost, 0, nb, s) != cudaSuccess) ||
            (dpre && cudaMemsetAsync(dpre, 0, nb, s) != cudaSuccess))
            return norm_fail(LIFB_ERR_CUDA, what, "memset failed");
        return LIFB_OK;
    }
    a.dxo = dxo;
    a.dn = dn;
    a.sdx = dxo_stride;
    a.sdn = dn_stride;
    a.dx = dx;
    a.dh = dh;
    a.dgate = dgate;
    if (!a.x || !a.rstd || (a.h && !a.post) || (dn && !a.pre) || (p->gate_cols && !p->gate) || (!dxo && !dn))
        return norm_fail(LIFB_ERR_INVALID_ARGUMENT, what, "null pointer");
    if (weights && (!workspace || !aligned16(workspace) || workspace_bytes < lifb_norm_gate_bwd_workspace_bytes(a.R, a.D, p->dtype)))
        return norm_fail(LIFB_ERR_WORKSPACE, what, "workspace missing, misaligned or too small");
    a.part = weights ? (float *)workspace : nullptr;
    const bool gate = a.gate && !a.gate_row;
    const int elem = (int)dtype_bytes(p->dtype);
    const int vec = norm_vec(elem, a.D, {a.sx, dxo ? a.sdx : 0, dn ? a.sdn : 0, a.h ? a.sh : 0, gate ? a.sg : 0},
                             {a.x, dx, dh, dxo, dn, a.h, gate ? a.gate : nullptr, gate ? dgate : nullptr});
    NormShape sh;
    if (!norm_shape(a.D, vec, elem, true, sh))
        return norm_fail(LIFB_ERR_UNSUPPORTED, what, "rows longer than 8192 elements");
    bool ok = false;
    LIFB_BY_DTYPE(p->dtype, T, ok = norm_run<T>(true, a, sh, s));
    if (ok && weights) {
        const int64_t parts = norm_blocks(sh, a.R, true);
        const unsigned blocks = (unsigned)((2 * a.D + 31) / 32);
        count_launches(1);
        LIFB_BY_DTYPE(p->dtype, T,
                      (k_norm_weight_grads<T><<<blocks, 32 * kNgReduceRows, 0, s>>>((const float *)workspace, parts,
                                                                                 a.D, dpost, dpre, a.w_f32)));
    }
    if (cudaGetLastError() != cudaSuccess || !ok) return norm_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}
