// Embedding with scaling, and its weight gradient by sorted tokens.
//
//   forward   y_i = scale * W[token_i]            (0 where token_i < 0)
//   gradient  dW[v] = scale * sum_{i: token_i = v} dy_i
//
// Both are bound by memory: the forward reads at most n rows and writes n, the
// gradient reads n rows and writes all V.  The gradient's sums run in an order
// that the tokens alone fix, so it gives the same bits each time: the token
// positions are sorted by token (a stable radix sort: digits of 8 to 10 bits, one
// counting and one placing launch a digit, one alone for up to kEmMinTile tokens), the sorted positions are
// cut into pieces of kEmPiece, and a piece adds its rows one after another in
// fp32.  A token whose positions lie within a piece is finished there; one that
// reaches over a piece's edge leaves that piece's part (fp32) to a last launch
// that joins the parts in order.  Rows of tokens that do not occur are zeroed by
// further blocks of the summing launch, so dW is written exactly once.
// Measured: 65536 tokens of 700, 256 wide in fp32: forward 17 us, sorting 25 us, sums
// 17 us, joins 6 us; 32768 of 50001, 1024 wide in bf16: 19, 21, 28 and 14 us.  Sorting is
// a chain of short launches, bound by latency; the sums by memory (10 us and 26 us of it).
#include <algorithm>

#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"
#include "tma.cuh"

namespace lifb {

namespace {

constexpr int kEmThreads = 256;
constexpr int kEmWarps = kEmThreads / 32;
constexpr int kEmMaxBits = 10;       // digit size: at most 1024 bins, 4 a thread
constexpr int kEmMinBits = 8;        // and at least 256, one a thread
// Sorting blocks: each reads the counts of all of them, from the same lines of L2 (64
// blocks of 1024 digits: 27 us of it), so few, and more only where tokens are many.
constexpr int kEmBlocks = 32, kEmBlocksMany = 64;
constexpr int64_t kEmMany = 1 << 17;
constexpr int kEmMinTile = 1024;     // tokens a sorting block takes at least
constexpr int kEmRows = 4;           // rows of the forward a thread
constexpr int kEmPiece = 64;         // sorted positions summed by one block

struct EmbedPlan {
    int bits, passes, radix_bits, blocks;
    int64_t tile, pieces;
};

EmbedPlan plan_of(int64_t n, int64_t V)
{
    EmbedPlan p;
    p.bits = 1;  // keys 0..V: V marks tokens without a row
    while ((int64_t(1) << p.bits) <= V) p.bits++;
    p.passes = (p.bits + kEmMaxBits - 1) / kEmMaxBits;
    p.radix_bits = std::max(kEmMinBits, (p.bits + p.passes - 1) / p.passes);
    const int most = n > kEmMany ? kEmBlocksMany : kEmBlocks;
    p.tile = std::max<int64_t>(kEmMinTile, (n + most - 1) / most);
    p.tile = (p.tile + kEmThreads - 1) / kEmThreads * kEmThreads;
    p.blocks = (int)((n + p.tile - 1) / p.tile);
    p.pieces = (n + kEmPiece - 1) / kEmPiece;
    return p;
}

struct EmbedWs {
    int32_t *key[2], *pos[2];
    int32_t *counts;
    uint8_t *present;
    float *head, *tail;
    size_t bytes;
};

EmbedWs carve(void *base, int64_t n, int64_t V, int64_t D)
{
    const EmbedPlan p = plan_of(n, V);
    EmbedWs w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        void *r = (char *)base + at;
        at += (bytes + 255) & ~(size_t)255;
        return r;
    };
    for (int i = 0; i < 2; i++) {
        w.key[i] = (int32_t *)take(n * 4);
        w.pos[i] = (int32_t *)take(n * 4);
    }
    w.counts = (int32_t *)take((size_t)p.blocks * (1 << p.radix_bits) * 4);
    w.present = (uint8_t *)take(V);
    w.head = (float *)take(p.pieces * D * 4);
    w.tail = (float *)take(p.pieces * D * 4);
    w.bytes = at;
    return w;
}

}  // namespace

// y = scale * W[token]: a block has blockDim.x vectors of VEC columns by blockDim.y
// rows, kEmRows of them a thread (their loads in flight together).  A token past the
// table gives zeros and sets the device status.
template <typename T, typename Tok, int VEC>
__global__ void __launch_bounds__(256) k_embed_fwd(const Tok *__restrict__ tokens, const T *__restrict__ W,
                                                   T *__restrict__ Y, int64_t n, int64_t V, int64_t D,
                                                   int64_t w_stride, float scale, int *status)
{
    const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int64_t r0 = (int64_t)blockIdx.x * blockDim.y * kEmRows + threadIdx.y;
    int64_t tok[kEmRows];
#pragma unroll
    for (int i = 0; i < kEmRows; i++) {
        const int64_t r = r0 + (int64_t)i * blockDim.y;
        tok[i] = r < n ? (int64_t)tokens[r] : -1;
        if (tok[i] >= V) {
            if (c == 0) atomicExch(status, kStatusTokenRange);
            tok[i] = -1;
        }
    }
    if (c >= D) return;
    float x[kEmRows][VEC];
#pragma unroll
    for (int i = 0; i < kEmRows; i++) {
#pragma unroll
        for (int e = 0; e < VEC; e++) x[i][e] = 0.0f;
        if (tok[i] >= 0) load_f32(W + tok[i] * w_stride + c, x[i]);
    }
#pragma unroll
    for (int i = 0; i < kEmRows; i++) {
        const int64_t r = r0 + (int64_t)i * blockDim.y;
#pragma unroll
        for (int e = 0; e < VEC; e++) x[i][e] *= scale;
        if (r < n) store_f32(Y + r * D + c, x[i]);
    }
}

// A token's key: itself, or V where it has no row.
template <typename Tok>
__device__ __forceinline__ int32_t embed_key(const Tok *tokens, int64_t i, int64_t V, int *status)
{
    const int64_t tok = (int64_t)tokens[i];
    if (tok >= V) atomicExch(status, kStatusTokenRange);
    return tok >= 0 && tok < V ? (int32_t)tok : (int32_t)V;
}

// Counts the digits of each block's tokens: counts[block][digit].  The first
// digit's launch also makes the keys and clears `present`.
template <typename Tok, bool FIRST>
__global__ void __launch_bounds__(kEmThreads)
    k_embed_count(const Tok *__restrict__ tokens, int32_t *__restrict__ key, int32_t *__restrict__ counts,
                  uint8_t *__restrict__ present, int64_t n, int64_t V, int64_t tile, int shift, int radix_bits,
                  int *status)
{
    __shared__ int32_t hist[1 << kEmMaxBits];
    const int radix = 1 << radix_bits;
    for (int d = threadIdx.x; d < radix; d += kEmThreads) hist[d] = 0;
    if (FIRST)
        for (int64_t v = (int64_t)blockIdx.x * kEmThreads + threadIdx.x; v < V; v += (int64_t)gridDim.x * kEmThreads)
            present[v] = 0;
    __syncthreads();
    const int64_t i0 = blockIdx.x * tile, i1 = min(n, i0 + tile);
#pragma unroll 4
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kEmThreads) {
        int32_t k;
        if (FIRST) {
            k = embed_key(tokens, i, V, status);
            key[i] = k;
        } else {
            k = key[i];
        }
        atomicAdd(&hist[(k >> shift) & (radix - 1)], 1);  // integers: the order does not matter
    }
    __syncthreads();
    for (int d = threadIdx.x; d < radix; d += kEmThreads) counts[(int64_t)blockIdx.x * radix + d] = hist[d];
}

// Places each block's tokens, in order, at their digit's place: the number of
// smaller digits, of this digit in earlier blocks, in earlier warps of the
// block (each warp owns a contiguous part of the tile), and before it in the warp.
// PER digits a thread.  ALONE: one block has all tokens; it counts for itself (and in
// the first digit's launch makes the keys and clears `present`).
template <typename Tok, int PER, bool FIRST, bool ALONE>
__global__ void __launch_bounds__(kEmThreads)
    k_embed_place(const Tok *__restrict__ tokens, const int32_t *__restrict__ key, const int32_t *__restrict__ pos,
                  int32_t *__restrict__ key_out, int32_t *__restrict__ pos_out, const int32_t *__restrict__ counts,
                  uint8_t *__restrict__ present, int64_t n, int64_t V, int64_t tile, int shift, int last, int *status)
{
    constexpr int radix = PER * kEmThreads;
    extern __shared__ int32_t em_smem[];
    int32_t *whist = em_smem;  // [warps][radix]
    __shared__ int32_t warp_sum[kEmWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto key_at = [&](int64_t i) {
        if constexpr (FIRST && ALONE) return embed_key(tokens, i, V, status);
        else return key[i];
    };
    for (int i = tid; i < kEmWarps * radix; i += kEmThreads) whist[i] = 0;
    if (FIRST && ALONE)
        for (int64_t v = tid; v < V; v += kEmThreads) present[v] = 0;
    __syncthreads();

    // digits of each warp's part
    const int64_t part = tile / kEmWarps;  // a multiple of 32
    const int64_t i0 = blockIdx.x * tile + warp * part, i1 = min(n, i0 + part);
    int32_t *wh = whist + warp * radix;
    constexpr int U = 8;  // tokens of a lane loaded together
    int32_t k8[U];
    auto load_keys = [&](int64_t i) {
#pragma unroll
        for (int j = 0; j < U; j++) k8[j] = i + 32 * j + lane < i1 ? key_at(i + 32 * j + lane) : -1;
    };
    for (int64_t i = i0; i < i1; i += 32 * U) {
        load_keys(i);
#pragma unroll
        for (int j = 0; j < U; j++)
            if (k8[j] >= 0) atomicAdd(&wh[(k8[j] >> shift) & (radix - 1)], 1);
    }

    // counts of this thread's digits in all blocks and in the earlier ones
    struct alignas(4 * PER) Counts {
        int32_t c[PER];
    };
    Counts total = {}, before = {};
    if (ALONE) {
        __syncthreads();
        for (int w = 0; w < kEmWarps; w++)
#pragma unroll
            for (int e = 0; e < PER; e++) total.c[e] += whist[w * radix + tid * PER + e];
    } else {
        const Counts *at = reinterpret_cast<const Counts *>(counts) + tid;
#pragma unroll 8
        for (int b = 0; b < (int)gridDim.x; b++) {
            const Counts x = at[(int64_t)b * kEmThreads];
#pragma unroll
            for (int e = 0; e < PER; e++) {
                total.c[e] += x.c[e];
                if (b < (int)blockIdx.x) before.c[e] += x.c[e];
            }
        }
    }
    int32_t mine = 0;
#pragma unroll
    for (int e = 0; e < PER; e++) mine += total.c[e];
    int32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t up = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int32_t start = incl - mine;
    for (int w = 0; w < warp; w++) start += warp_sum[w];
    // each warp's first place of each digit
#pragma unroll
    for (int e = 0; e < PER; e++) {
        const int d = tid * PER + e;
        int32_t s = start + before.c[e];
        start += total.c[e];
        for (int w = 0; w < kEmWarps; w++) {
            const int32_t c = whist[w * radix + d];
            whist[w * radix + d] = s;
            s += c;
        }
    }
    __syncthreads();
    for (int64_t i = i0; i < i1; i += 32 * U) {  // uniform over the warp
        if (i1 - i0 > 32 * U) load_keys(i);      // else still there
        int32_t from[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int64_t at = i + 32 * j + lane;
            from[j] = FIRST ? (int32_t)at : k8[j] >= 0 ? pos[at] : 0;
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            const bool on = k8[j] >= 0;
            const int d = on ? (k8[j] >> shift) & (radix - 1) : -1;
            const unsigned same = __match_any_sync(~0u, d);
            const int rank = __popc(same & ((1u << lane) - 1));
            int32_t at = 0;
            if (on) at = wh[d] + rank;
            __syncwarp();
            if (on && rank == 0) wh[d] += __popc(same);
            __syncwarp();
            if (on) {
                key_out[at] = k8[j];
                pos_out[at] = from[j];
                if (last && k8[j] < V) present[k8[j]] = 1;
            }
        }
    }
}

// Blocks [0, pieces): sums of one piece of sorted positions, VEC columns a
// thread.  Blocks past them: zeros for the rows of tokens that do not occur.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    k_embed_sum(const int32_t *__restrict__ key, const int32_t *__restrict__ pos, const T *__restrict__ dY,
                T *__restrict__ dW, float *__restrict__ head, float *__restrict__ tail,
                const uint8_t *__restrict__ present, int64_t n, int64_t V, int64_t D, int64_t dy_stride,
                int64_t pieces, float scale)
{
    __shared__ int32_t s_key[kEmPiece + 2], s_pos[kEmPiece];
    const int tid = threadIdx.x;
    if (blockIdx.x >= pieces) {
        // 32 rows' marks at a time
        const int64_t per = D / VEC, nz = gridDim.x - pieces, z = blockIdx.x - pieces;
        const int lane = tid & 31;
        float zero[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) zero[i] = 0.0f;
        for (int64_t v0 = z * 32; v0 < V; v0 += nz * 32) {
            unsigned absent = __ballot_sync(~0u, v0 + lane < V && !present[min(v0 + lane, V - 1)]);
            while (absent) {
                const int64_t v = v0 + __ffs(absent) - 1;
                absent &= absent - 1;
                for (int64_t c = tid; c < per; c += blockDim.x) store_f32(dW + v * D + c * VEC, zero);
            }
        }
        return;
    }
    const int64_t p = blockIdx.x, i0 = p * kEmPiece;
    const int m = (int)min((int64_t)kEmPiece, n - i0);
    for (int i = tid; i < m + 2; i += blockDim.x) {  // the keys beside the piece too; -1 outside
        const int64_t at = i0 + i - 1;
        s_key[i] = at >= 0 && at < n ? key[at] : -1;
        if (i < m) s_pos[i] = pos[i0 + i];
    }
    __syncthreads();
    const bool from_before = s_key[0] == s_key[1];
    for (int64_t c = (int64_t)tid * VEC; c < D; c += (int64_t)blockDim.x * VEC) {
        float acc[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
        int first = 0;  // where the current token's run starts in the piece
        constexpr int U = 16;  // rows in flight
        for (int i = 0; i < m; i += U) {
            Pack<T, VEC> raw[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i + u < m && s_key[i + u + 1] < V) raw[u].load(dY + (int64_t)s_pos[i + u] * dy_stride + c);
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (i + u >= m) break;
                const int32_t k = s_key[i + u + 1];
                if (k >= V) break;  // the tokens without a row are last
                float x[VEC];
                raw[u].get(x);
#pragma unroll
                for (int e = 0; e < VEC; e++) acc[e] += x[e];
                if (s_key[i + u + 2] != k || i + u == m - 1) {  // the run's end, or the piece's
                    if (first == 0 && from_before) {
                        store_f32(head + p * D + c, acc);
                    } else if (i + u == m - 1 && s_key[i + u + 2] == k) {
                        store_f32(tail + p * D + c, acc);
                    } else {
                        float y[VEC];
#pragma unroll
                        for (int e = 0; e < VEC; e++) y[e] = acc[e] * scale;
                        store_f32(dW + (int64_t)k * D + c, y);
                    }
#pragma unroll
                    for (int e = 0; e < VEC; e++) acc[e] = 0.0f;
                    first = i + u + 1;
                }
            }
        }
    }
}

// Joins the parts of a token that reaches over pieces' edges, in order; the
// piece where its run starts does it.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    k_embed_join(const int32_t *__restrict__ key, T *__restrict__ dW, const float *__restrict__ head,
                 const float *__restrict__ tail, int64_t n, int64_t V, int64_t D, int64_t pieces, float scale)
{
    const int64_t p = blockIdx.x, end = (p + 1) * kEmPiece;
    if (end >= n) return;
    const int32_t k = key[end - 1], after = key[end], before = p > 0 ? key[p * kEmPiece - 1] : -1;
    if (k >= V || after != k) return;  // nothing goes on past this piece
    if (before == k && key[p * kEmPiece] == k) return;  // it starts in an earlier piece
    __shared__ int64_t s_last;
    if (threadIdx.x < 32) {
        // The last piece that it reaches: the first one after p whose end is not k, if that
        // begins with k (32 of them tested at a time).
        int64_t lo = p + 1, hi = pieces - 1;
        while (lo < hi) {
            const int64_t step = (hi - lo + 31) / 32, at = lo + threadIdx.x * step;
            const unsigned past = __ballot_sync(~0u, at >= hi || key[min(n, (at + 1) * kEmPiece) - 1] != k);
            const int first = __ffs(past) - 1;  // lane 31 is at or past hi only if step covers it
            if (past == 0) {
                lo = lo + 31 * step + 1;
            } else {
                const int64_t f = min(hi, lo + first * step);
                lo = first == 0 ? lo : lo + (first - 1) * step + 1;
                hi = f;
            }
        }
        if (threadIdx.x == 0) s_last = key[lo * kEmPiece] == k ? lo : lo - 1;
    }
    __syncthreads();
    const int64_t last = s_last;
    for (int64_t c = (int64_t)threadIdx.x * VEC; c < D; c += (int64_t)blockDim.x * VEC) {
        float acc[VEC];
        load_f32(tail + p * D + c, acc);
#pragma unroll 8
        for (int64_t q = p + 1; q <= last; q++) {
            float x[VEC];
            load_f32(head + q * D + c, x);
#pragma unroll
            for (int e = 0; e < VEC; e++) acc[e] += x[e];
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) acc[e] *= scale;
        store_f32(dW + (int64_t)k * D + c, acc);
    }
}

namespace {

unsigned round_threads(int64_t want)
{
    return (unsigned)std::min<int64_t>(256, std::max<int64_t>(32, (want + 31) / 32 * 32));
}

template <typename T, typename Tok, int VEC>
void embed_fwd(const void *tokens, const void *W, void *Y, int64_t n, int64_t V, int64_t D, int64_t w_stride,
               float scale, cudaStream_t s)
{
    const int64_t vecs = (D + VEC - 1) / VEC;
    const unsigned x = vecs >= 256 ? 256 : round_threads(vecs), y = 256 / x;
    const dim3 grid((unsigned)((n + y * kEmRows - 1) / (y * kEmRows)), (unsigned)((vecs + x - 1) / x));
    count_launches(1);
    k_embed_fwd<T, Tok, VEC><<<grid, dim3(x, y), 0, s>>>((const Tok *)tokens, (const T *)W, (T *)Y, n, V, D, w_stride,
                                                         scale, device_status_ptr());
}

template <typename T, int VEC>
void embed_sum(const EmbedWs &w, int last, const EmbedPlan &p, const void *dY, void *dW, int64_t n, int64_t V,
               int64_t D, int64_t dy_stride, float scale, cudaStream_t s)
{
    const unsigned threads = round_threads((D + VEC - 1) / VEC);
    const int64_t zero_blocks = std::min<int64_t>((V + 31) / 32, 148 * 8);
    count_launches(2);
    k_embed_sum<T, VEC><<<(unsigned)(p.pieces + zero_blocks), threads, 0, s>>>(
        w.key[last], w.pos[last], (const T *)dY, (T *)dW, w.head, w.tail, w.present, n, V, D, dy_stride, p.pieces,
        scale);
    k_embed_join<T, VEC><<<(unsigned)p.pieces, threads, 0, s>>>(w.key[last], (T *)dW, w.head, w.tail, n, V, D,
                                                                p.pieces, scale);
}

template <typename Tok, int PER>
int embed_sort(const EmbedWs &w, const EmbedPlan &p, const void *tokens, int64_t n, int64_t V, cudaStream_t s)
{
    const size_t smem = (size_t)kEmWarps * (1 << p.radix_bits) * 4;  // 32 KB at most
    int cur = 0;
    for (int pass = 0; pass < p.passes; pass++) {
        const int shift = pass * p.radix_bits;
        const bool first = pass == 0, alone = p.blocks == 1;
        const Tok *tok = (const Tok *)tokens;
        if (!alone) {
            count_launches(1);
            auto count = first ? k_embed_count<Tok, true> : k_embed_count<Tok, false>;
            count<<<p.blocks, kEmThreads, 0, s>>>(tok, w.key[cur], w.counts, w.present, n, V, p.tile, shift,
                                                  p.radix_bits, device_status_ptr());
        }
        auto place = first ? (alone ? k_embed_place<Tok, PER, true, true> : k_embed_place<Tok, PER, true, false>)
                           : (alone ? k_embed_place<Tok, PER, false, true> : k_embed_place<Tok, PER, false, false>);
        count_launches(1);
        place<<<p.blocks, kEmThreads, smem, s>>>(tok, w.key[cur], w.pos[cur], w.key[cur ^ 1], w.pos[cur ^ 1], w.counts,
                                                 w.present, n, V, p.tile, shift, pass == p.passes - 1,
                                                 device_status_ptr());
        cur ^= 1;
    }
    return cur;
}

template <typename Tok>
int embed_sort(const EmbedWs &w, const EmbedPlan &p, const void *tokens, int64_t n, int64_t V, cudaStream_t s)
{
    return p.radix_bits == 8   ? embed_sort<Tok, 1>(w, p, tokens, n, V, s)
           : p.radix_bits == 9 ? embed_sort<Tok, 2>(w, p, tokens, n, V, s)
                               : embed_sort<Tok, 4>(w, p, tokens, n, V, s);
}

int embed_check(const char *what, const void *tokens, int token_bytes, const void *a, const void *b, int64_t n,
                int64_t V, int64_t D, int64_t stride, int dtype)
{
    auto bad = [&](int status, const char *why) {
        char msg[160];
        snprintf(msg, sizeof msg, "%s: %s", what, why);
        set_last_error(msg);
        return status;
    };
    if (n < 0 || V < 0 || D < 0) return bad(LIFB_ERR_INVALID_ARGUMENT, "negative shape");
    if (!dtype_bytes(dtype)) return bad(LIFB_ERR_INVALID_ARGUMENT, "unknown dtype");
    if (token_bytes != 4 && token_bytes != 8) return bad(LIFB_ERR_INVALID_ARGUMENT, "tokens have 4 or 8 bytes");
    if (n >= (int64_t(1) << 31) - (1 << 20) || V >= (int64_t(1) << 30) || D >= (int64_t(1) << 24))
        return bad(LIFB_ERR_UNSUPPORTED, "needs n < 2^31 - 2^20, V < 2^30, D < 2^24");
    if (stride < D) return bad(LIFB_ERR_INVALID_ARGUMENT, "row stride below the row's length");
    if ((n > 0 && !tokens) || (n > 0 && D > 0 && !a) || (n > 0 && D > 0 && V > 0 && !b))
        return bad(LIFB_ERR_INVALID_ARGUMENT, "null pointer");
    return LIFB_OK;
}

int embed_done(const char *what)
{
    if (cudaGetLastError() != cudaSuccess) {
        char msg[96];
        snprintf(msg, sizeof msg, "%s: launch failed", what);
        set_last_error(msg);
        return LIFB_ERR_CUDA;
    }
    set_last_error("");
    return LIFB_OK;
}

}  // namespace

}  // namespace lifb

extern "C" int lifb_embed_fwd(const void *tokens, int token_bytes, const void *W, void *Y, int64_t n, int64_t V,
                              int64_t D, int64_t w_stride, float scale, int dtype, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_embed_fwd");
    if (int st = embed_check("lifb_embed_fwd", tokens, token_bytes, Y, W, n, V, D, w_stride, dtype)) return st;
    if (n == 0 || D == 0) return LIFB_OK;
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t vec = 16 / dtype_bytes(dtype);
    const bool wide = D % vec == 0 && w_stride % vec == 0 && aligned16(W) && aligned16(Y);
    LIFB_BY_DTYPE(dtype, T, {
        constexpr int VEC = 16 / sizeof(T);
        if (token_bytes == 8) {
            if (wide) embed_fwd<T, int64_t, VEC>(tokens, W, Y, n, V, D, w_stride, scale, s);
            else embed_fwd<T, int64_t, 1>(tokens, W, Y, n, V, D, w_stride, scale, s);
        } else {
            if (wide) embed_fwd<T, int32_t, VEC>(tokens, W, Y, n, V, D, w_stride, scale, s);
            else embed_fwd<T, int32_t, 1>(tokens, W, Y, n, V, D, w_stride, scale, s);
        }
    });
    return embed_done("lifb_embed_fwd");
}

extern "C" size_t lifb_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D)
{
    if (n <= 0 || V <= 0 || D <= 0 || V >= (int64_t(1) << 30)) return 0;
    return lifb::carve(nullptr, n, V, D).bytes;
}

extern "C" int lifb_embed_bwd(const void *tokens, int token_bytes, const void *dY, void *dW, int64_t n, int64_t V,
                              int64_t D, int64_t dy_stride, float scale, int dtype, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    using namespace lifb;
    LIFB_RANGE("lifb_embed_bwd");
    if (int st = embed_check("lifb_embed_bwd", tokens, token_bytes, dW, dY, n, V, D, dy_stride, dtype)) return st;
    if (V == 0 || D == 0) return LIFB_OK;
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        if (!dW) {
            set_last_error("lifb_embed_bwd: null pointer");
            return LIFB_ERR_INVALID_ARGUMENT;
        }
        if (cudaMemsetAsync(dW, 0, (size_t)V * D * dtype_bytes(dtype), s) != cudaSuccess) {
            set_last_error("lifb_embed_bwd: memset failed");
            return LIFB_ERR_CUDA;
        }
        return LIFB_OK;
    }
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < lifb_embed_bwd_workspace_bytes(n, V, D)) {
        set_last_error("lifb_embed_bwd: workspace missing, misaligned or too small");
        return LIFB_ERR_WORKSPACE;
    }
    const EmbedPlan p = plan_of(n, V);
    const EmbedWs w = carve(workspace, n, V, D);
    const int last = token_bytes == 8 ? embed_sort<int64_t>(w, p, tokens, n, V, s) : embed_sort<int32_t>(w, p, tokens, n, V, s);
    const int64_t vec = 16 / dtype_bytes(dtype);
    const bool wide = D % vec == 0 && dy_stride % vec == 0 && aligned16(dY) && aligned16(dW);
    LIFB_BY_DTYPE(dtype, T, {
        constexpr int VEC = 16 / sizeof(T);
        // 8 elements of a 16-bit type make 32 bytes of fp32 partial sums: stored as two vectors
        if (wide) embed_sum<T, VEC>(w, last, p, dY, dW, n, V, D, dy_stride, scale, s);
        else embed_sum<T, 1>(w, last, p, dY, dW, n, V, D, dy_stride, scale, s);
    });
    return embed_done("lifb_embed_bwd");
}
