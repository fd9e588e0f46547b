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
// its rows' parts of dpre and dpost there, in row order; the groups' sums (fp32)
// are added by a second launch in a fixed order.
#include <algorithm>

#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"

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
    float *part;  // [blocks * groups][2][D]
    int64_t R, D;
    float scale, eps;
    int act, gate_row, w_f32;
};

}  // namespace

// Sums NV values over the TPR threads of a row; every thread gets them.
// `sh`: NV * warps of the block floats, used twice alternately by `flip`.
template <int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], int tpr, float *sh, int &flip)
{
    const int in_warp = tpr < 32 ? tpr : 32;
    for (int o = in_warp >> 1; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < NV; i++) v[i] += __shfl_xor_sync(~0u, v[i], o);
    }
    if (tpr > 32) {
        // rows of one block reduce in lockstep: every group makes the same calls
        const int warp = threadIdx.x >> 5, wpr = tpr >> 5, w0 = warp / wpr * wpr;
        float *buf = sh + flip * NV * 32;
        flip ^= 1;
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) buf[i * 32 + warp] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float s = 0.0f;
            for (int w = 0; w < wpr; w++) s += buf[i * 32 + w0 + w];
            v[i] = s;
        }
    }
}

__device__ __forceinline__ float act_value(int act, float g)
{
    if (act == kActLinear) return g;
    const float sg = 1.0f / (1.0f + expf(-g));
    return act == kActSilu ? g * sg : sg;
}

// act(g) and act'(g)
__device__ __forceinline__ void act_grad(int act, float g, float &a, float &da)
{
    if (act == kActLinear) {
        a = g;
        da = 1.0f;
        return;
    }
    const float sg = 1.0f / (1.0f + expf(-g));
    a = act == kActSilu ? g * sg : sg;
    da = act == kActSilu ? sg * (1.0f + g * (1.0f - sg)) : sg * (1.0f - sg);
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void *w, int f32, int64_t c, float (&x)[VEC])
{
    if (f32) {
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = ((const float *)w)[c + e];
    } else {
        load_f32((const T *)w + c, x);
    }
}

template <typename T, int VEC, int NIT, int MAXT>
__global__ void __launch_bounds__(MAXT)
    k_norm_fwd(const __grid_constant__ NormArgs a, int tpr)
{
    __shared__ float sh[2 * 32];
    int flip = 0;
    const int lane = threadIdx.x & (tpr - 1);
    const int64_t groups = blockDim.x / tpr, g = threadIdx.x / tpr;
    const float inv_d = 1.0f / (float)a.D;
    float post[NIT][VEC], pre[NIT][VEC];
#pragma unroll
    for (int i = 0; i < NIT; i++) {
        const int64_t c = ((int64_t)i * tpr + lane) * VEC;
        if (c < a.D) {
            if (a.h) load_weight<T, VEC>(a.post, a.w_f32, c, post[i]);
            if (a.n) load_weight<T, VEC>(a.pre, a.w_f32, c, pre[i]);
        }
    }
    // every group of a block makes the same number of rounds
    for (int64_t r0 = blockIdx.x * groups; r0 < a.R; r0 += gridDim.x * groups) {
        const int64_t r = r0 + g;
        const bool on = r < a.R;
        float x[NIT][VEC], h[NIT][VEC], gt[NIT][VEC];
        float ss[1] = {0.0f};
        float grow = 0.0f;
        if (on && a.h && a.gate && a.gate_row) grow = to_f32(((const T *)a.gate)[r * a.sg]);
#pragma unroll
        for (int i = 0; i < NIT; i++) {
            const int64_t c = ((int64_t)i * tpr + lane) * VEC;
            const bool in = on && c < a.D;
#pragma unroll
            for (int e = 0; e < VEC; e++) x[i][e] = h[i][e] = gt[i][e] = 0.0f;
            if (in) {
                load_f32((const T *)a.x + r * a.sx + c, x[i]);
                if (a.h) {
                    load_f32((const T *)a.h + r * a.sh + c, h[i]);
                    if (a.gate && !a.gate_row) load_f32((const T *)a.gate + r * a.sg + c, gt[i]);
                }
            }
        }
        if (a.h) {
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) ss[0] += h[i][e] * h[i][e];
            row_sum(ss, tpr, sh, flip);
            const float rh = rsqrtf(ss[0] * inv_d + a.eps);
            if (on && lane == 0 && a.rstd) a.rstd[r] = rh;
            const float arow = a.gate && a.gate_row ? act_value(a.act, grow) : 1.0f;
#pragma unroll
            for (int i = 0; i < NIT; i++) {
                const int64_t c = ((int64_t)i * tpr + lane) * VEC;
                if (on && c < a.D) {
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const float av = a.gate && !a.gate_row ? act_value(a.act, gt[i][e]) : arow;
                        x[i][e] += a.scale * (av * (h[i][e] * rh * post[i][e]));
                    }
                    store_f32((T *)a.xo + r * a.D + c, x[i]);
                }
            }
        }
        if (a.n) {
            ss[0] = 0.0f;
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) ss[0] += x[i][e] * x[i][e];
            row_sum(ss, tpr, sh, flip);
            const float rx = rsqrtf(ss[0] * inv_d + a.eps);
            if (on && lane == 0 && a.rstd) a.rstd[a.R + r] = rx;
#pragma unroll
            for (int i = 0; i < NIT; i++) {
                const int64_t c = ((int64_t)i * tpr + lane) * VEC;
                if (on && c < a.D) {
                    float y[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; e++) y[e] = x[i][e] * rx * pre[i][e];
                    store_f32((T *)a.n + r * a.D + c, y);
                }
            }
        }
    }
}

template <typename T, int VEC, int NIT, int MAXT>
__global__ void __launch_bounds__(MAXT)
    k_norm_bwd(const __grid_constant__ NormArgs a, int tpr)
{
    __shared__ float sh[2 * 2 * 32];
    int flip = 0;
    const int lane = threadIdx.x & (tpr - 1);
    const int64_t groups = blockDim.x / tpr, g = threadIdx.x / tpr;
    const float inv_d = 1.0f / (float)a.D;
    float post[NIT][VEC], pre[NIT][VEC], dpost[NIT][VEC], dpre[NIT][VEC];
#pragma unroll
    for (int i = 0; i < NIT; i++) {
        const int64_t c = ((int64_t)i * tpr + lane) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; e++) dpost[i][e] = dpre[i][e] = post[i][e] = pre[i][e] = 0.0f;
        if (c < a.D) {
            if (a.h) load_weight<T, VEC>(a.post, a.w_f32, c, post[i]);
            if (a.dn) load_weight<T, VEC>(a.pre, a.w_f32, c, pre[i]);
        }
    }
    for (int64_t r0 = blockIdx.x * groups; r0 < a.R; r0 += gridDim.x * groups) {
        const int64_t r = r0 + g;
        const bool on = r < a.R;
        // t: dx', then the gradient of x'; x: x, then x'; hh: h, then h r(h)
        float t[NIT][VEC], x[NIT][VEC], hh[NIT][VEC], gt[NIT][VEC], u[NIT][VEC];
        float rh = 0.0f, rx = 0.0f, grow = 0.0f;
        if (on) {
            if (a.h) rh = a.rstd[r];
            if (a.dn) rx = a.rstd[a.R + r];
            if (a.h && a.gate && a.gate_row) grow = to_f32(((const T *)a.gate)[r * a.sg]);
        }
#pragma unroll
        for (int i = 0; i < NIT; i++) {
            const int64_t c = ((int64_t)i * tpr + lane) * VEC;
            const bool in = on && c < a.D;
#pragma unroll
            for (int e = 0; e < VEC; e++) t[i][e] = x[i][e] = hh[i][e] = gt[i][e] = u[i][e] = 0.0f;
            if (in) {
                if (a.dxo) load_f32((const T *)a.dxo + r * a.sdx + c, t[i]);
                if (a.dn) {
                    load_f32((const T *)a.dn + r * a.sdn + c, u[i]);
                    load_f32((const T *)a.x + r * a.sx + c, x[i]);
                }
                if (a.h) {
                    load_f32((const T *)a.h + r * a.sh + c, hh[i]);
                    if (a.gate && !a.gate_row) load_f32((const T *)a.gate + r * a.sg + c, gt[i]);
                }
            }
        }
        float arow = 1.0f, darow = 0.0f;
        if (a.h && a.gate && a.gate_row) act_grad(a.act, grow, arow, darow);
        if (a.h) {
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const float av = a.gate && !a.gate_row ? act_value(a.act, gt[i][e]) : arow;
                    hh[i][e] *= rh;
                    x[i][e] += a.scale * (av * (hh[i][e] * post[i][e]));
                }
        }
        if (a.dn) {
            float m[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    x[i][e] *= rx;
                    dpre[i][e] += u[i][e] * x[i][e];
                    u[i][e] *= pre[i][e];
                    m[0] += u[i][e] * x[i][e];
                }
            row_sum(m, tpr, sh, flip);
            const float mu = m[0] * inv_d;
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) t[i][e] += rx * (u[i][e] - x[i][e] * mu);
        }
#pragma unroll
        for (int i = 0; i < NIT; i++) {
            const int64_t c = ((int64_t)i * tpr + lane) * VEC;
            if (on && c < a.D && a.dx) store_f32((T *)a.dx + r * a.D + c, t[i]);
        }
        if (a.h) {
            float m[2] = {0.0f, 0.0f};  // mean of w * hh; the row gate's sum of t * y
#pragma unroll
            for (int i = 0; i < NIT; i++)
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    float av = arow, da = 0.0f;
                    if (a.gate && !a.gate_row) act_grad(a.act, gt[i][e], av, da);
                    const float st = a.scale * t[i][e], ty = st * (hh[i][e] * post[i][e]);
                    gt[i][e] = ty * da;
                    m[1] += ty;
                    dpost[i][e] += st * av * hh[i][e];
                    t[i][e] = st * av * post[i][e];
                    m[0] += t[i][e] * hh[i][e];
                }
            row_sum(m, tpr, sh + 0, flip);
            const float mw = m[0] * inv_d;
#pragma unroll
            for (int i = 0; i < NIT; i++) {
                const int64_t c = ((int64_t)i * tpr + lane) * VEC;
                if (!(on && c < a.D)) continue;
                float d[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) d[e] = rh * (t[i][e] - hh[i][e] * mw);
                if (a.dh) store_f32((T *)a.dh + r * a.D + c, d);
                if (a.dgate && !a.gate_row) store_f32((T *)a.dgate + r * a.D + c, gt[i]);
            }
            if (a.dgate && a.gate_row && on && lane == 0) ((T *)a.dgate)[r] = from_f32<T>(m[1] * darow);
        }
    }
    if (!a.part) return;
    float *part = a.part + (blockIdx.x * groups + g) * 2 * a.D;
#pragma unroll
    for (int i = 0; i < NIT; i++) {
        const int64_t c = ((int64_t)i * tpr + lane) * VEC;
        if (c < a.D) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                part[c + e] = dpost[i][e];
                part[a.D + c + e] = dpre[i][e];
            }
        }
    }
}

// Adds the groups' parts column by column, in order: 32 columns a block, one
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

// A row that a warp can hold stays in one warp (no block barrier); a longer one
// takes a thread for each vector up to a block of kNgThreads, then more vectors
// a thread, then a block of kNgMaxThreads.
bool norm_shape(int64_t D, bool wide, int elem, NormShape &s)
{
    s.vec = wide ? 16 / elem : 1;
    const int64_t vecs = (D + s.vec - 1) / s.vec;
    const int most = kNgMaxElems / s.vec;
    auto spread = [&](int tpr) {
        s.tpr = tpr;
        s.nit = 1;
        while (s.nit < most && (int64_t)s.tpr * s.nit < vecs) s.nit *= 2;
        return (int64_t)s.tpr * s.nit >= vecs;
    };
    s.threads = kNgThreads;
    for (int tpr = 8; tpr < 32; tpr *= 2)
        if (tpr >= vecs) return spread(tpr);
    if (spread(32)) return true;
    for (int tpr = 64; tpr <= kNgThreads; tpr *= 2)
        if (tpr >= vecs) return spread(tpr);
    if (spread(kNgThreads)) return true;
    s.threads = kNgMaxThreads;
    return spread(kNgMaxThreads);
}

int64_t norm_blocks(const NormShape &s, int64_t R)
{
    const int64_t groups = s.threads / s.tpr;
    const int64_t per_sm = 1024 / s.threads;
    return std::max<int64_t>(1, std::min<int64_t>((R + groups - 1) / groups, kNgSms * per_sm));
}

template <typename T, int VEC, int NIT>
void norm_launch(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    const unsigned blocks = (unsigned)norm_blocks(sh, a.R);
    count_launches(1);
    if (sh.threads == kNgThreads) {
        if (bwd) k_norm_bwd<T, VEC, NIT, kNgThreads><<<blocks, kNgThreads, 0, s>>>(a, sh.tpr);
        else k_norm_fwd<T, VEC, NIT, kNgThreads><<<blocks, kNgThreads, 0, s>>>(a, sh.tpr);
    } else if constexpr (VEC * NIT == kNgMaxElems) {  // a block of a long row is full
        if (bwd) k_norm_bwd<T, VEC, NIT, kNgMaxThreads><<<blocks, kNgMaxThreads, 0, s>>>(a, sh.tpr);
        else k_norm_fwd<T, VEC, NIT, kNgMaxThreads><<<blocks, kNgMaxThreads, 0, s>>>(a, sh.tpr);
    }
}

template <typename T, int VEC>
void norm_pick(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    switch (sh.nit) {
        case 1: norm_launch<T, VEC, 1>(bwd, a, sh, s); break;
        case 2: norm_launch<T, VEC, 2>(bwd, a, sh, s); break;
        case 4:
            if constexpr (VEC <= 4) norm_launch<T, VEC, 4>(bwd, a, sh, s);
            break;
        case 8:
            if constexpr (VEC == 1) norm_launch<T, VEC, 8>(bwd, a, sh, s);
            break;
        default:
            if constexpr (VEC == 1) norm_launch<T, VEC, 16>(bwd, a, sh, s);
    }
}

template <typename T>
void norm_run(bool bwd, const NormArgs &a, const NormShape &sh, cudaStream_t s)
{
    constexpr int VEC = 16 / sizeof(T);
    if (sh.vec == VEC) norm_pick<T, VEC>(bwd, a, sh, s);
    else norm_pick<T, 1>(bwd, a, sh, s);
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
    const int64_t vec = 16 / dtype_bytes(p->dtype);
    bool wide = a.D % vec == 0 && a.sx % vec == 0 && aligned16(a.x) && aligned16(xo) && aligned16(n);
    if (a.h) wide = wide && a.sh % vec == 0 && aligned16(a.h) && aligned16(a.post);
    if (n) wide = wide && aligned16(a.pre);
    if (a.gate && !a.gate_row) wide = wide && a.sg % vec == 0 && aligned16(a.gate);
    NormShape sh;
    if (!norm_shape(a.D, wide, (int)dtype_bytes(p->dtype), sh))
        return norm_fail(LIFB_ERR_UNSUPPORTED, what, "rows longer than 8192 elements");
    LIFB_BY_DTYPE(p->dtype, T, norm_run<T>(false, a, sh, (cudaStream_t)stream));
    if (cudaGetLastError() != cudaSuccess) return norm_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}

extern "C" size_t lifb_norm_gate_bwd_workspace_bytes(int64_t R, int64_t D, int dtype)
{
    using namespace lifb;
    if (R <= 0 || D <= 0 || !dtype_bytes(dtype)) return 0;
    size_t most = 0;  // of the vector and the element form
    for (int wide = 0; wide < 2; wide++) {
        NormShape sh;
        if (norm_shape(D, wide != 0, (int)dtype_bytes(dtype), sh))
            most = std::max(most, (size_t)norm_blocks(sh, R) * (sh.threads / sh.tpr) * 2 * D * 4);
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
    if (a.R == 0 || a.D == 0) {
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
    if (weights && (!workspace || workspace_bytes < lifb_norm_gate_bwd_workspace_bytes(a.R, a.D, p->dtype)))
        return norm_fail(LIFB_ERR_WORKSPACE, what, "workspace missing or too small");
    a.part = weights ? (float *)workspace : nullptr;
    const int64_t vec = 16 / dtype_bytes(p->dtype);
    bool wide = a.D % vec == 0 && a.sx % vec == 0 && aligned16(a.x) && aligned16(dx) && aligned16(dh);
    if (dxo) wide = wide && dxo_stride % vec == 0 && aligned16(dxo);
    if (dn) wide = wide && dn_stride % vec == 0 && aligned16(dn) && aligned16(a.pre);
    if (a.h) wide = wide && a.sh % vec == 0 && aligned16(a.h) && aligned16(a.post);
    if (a.gate && !a.gate_row) wide = wide && a.sg % vec == 0 && aligned16(a.gate) && aligned16(dgate);
    NormShape sh;
    if (!norm_shape(a.D, wide, (int)dtype_bytes(p->dtype), sh))
        return norm_fail(LIFB_ERR_UNSUPPORTED, what, "rows longer than 8192 elements");
    LIFB_BY_DTYPE(p->dtype, T, norm_run<T>(true, a, sh, s));
    if (weights) {
        const int64_t parts = norm_blocks(sh, a.R) * (sh.threads / sh.tpr);
        const unsigned blocks = (unsigned)((2 * a.D + 31) / 32);
        count_launches(1);
        LIFB_BY_DTYPE(p->dtype, T,
                      (k_norm_weight_grads<T><<<blocks, 32 * kNgReduceRows, 0, s>>>((const float *)workspace, parts,
                                                                                 a.D, dpost, dpre, a.w_f32)));
    }
    if (cudaGetLastError() != cudaSuccess) return norm_fail(LIFB_ERR_CUDA, what, "launch failed");
    set_last_error("");
    return LIFB_OK;
}
