// Softmax cross entropy of a classifier over a large vocabulary, and its
// gradient, straight from the hidden states and the classifier's weights:
//
//     z_tv = alpha sum_h x_th w_vh,   lse_t = log sum_v exp z_tv,
//     loss_t = lse_t - z_t,label(t)
//     P_tv = gloss_t (softmax(z_t)_v - [v = label(t)]) + glse_t softmax(z_t)_v
//     gX = alpha P W,   gW = alpha P^T X + beta gW
//
// The logits are never kept.  The forward pass reduces them to one maximum and
// one sum per token and tile of the vocabulary in the epilogue of the product
// (product kernel: xent_kernel.hip.h); the backward pass computes them again,
// a piece of the vocabulary at a time, and keeps P of one piece while the two
// products that need it run.  Tokens without a target (their label is `ignore`
// or no row of the classifier) are left out at the start: the rows of X that
// count are gathered into a compact copy, every product runs over those rows
// only, and what the other rows of X hold never reaches a result.
//
// Every sum is made in a fixed order: the same call gives the same bits.
#include "internal.h"
#include "xent_kernel.hip.h"

#include <algorithm>
#include <cstdio>

using namespace ulmgpu;
using namespace ulmgpu::xent;

namespace ulmgpu {
namespace {

// ---------------------------------------------------------------------------
// small kernels around the products
// ---------------------------------------------------------------------------

struct TokenArgs {
    int tokens, vocab, ignore;
    const int *label;
    float *loss, *lse_out;              // forward: zeros for rows without a target (null: not wanted)
    int *count, *rows, *label_c;        // rows that count, in order, and their labels
    int *place;                         // backward: compact place of every row or -1
    const float *lse, *gloss, *glse;    // backward: gathered and combined
    float alpha;
    float *lse_c, *both_c, *gloss_c;
};

// The label of row t, or -1 if it is none.
__device__ __forceinline__ int target_of(const TokenArgs &g, int t)
{
    const int y = g.label[t];
    return y == g.ignore || y < 0 || y >= g.vocab ? -1 : y;
}

// Row t has label y and compact place c, or no target (y < 0).
__device__ __forceinline__ void note_row(const TokenArgs &g, int t, int y, int c)
{
    if (y >= 0) {
        g.rows[c] = t;
        g.label_c[c] = y;
        if (g.lse) {
            const float gl = g.gloss[t];
            g.lse_c[c] = g.lse[t];
            g.gloss_c[c] = g.alpha * gl;
            g.both_c[c] = g.alpha * (g.glse ? gl + g.glse[t] : gl);
        }
    } else if (g.loss) {
        g.loss[t] = 0.0f;
        g.lse_out[t] = 0.0f;
    }
    if (g.place) g.place[t] = y >= 0 ? c : -1;
}

// One workgroup: which rows have a target, in order.
__global__ void __launch_bounds__(1024) token_kernel(TokenArgs g)
{
    __shared__ int wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int done = 0;
    for (int t0 = 0; t0 < g.tokens; t0 += 1024) {
        const int t = t0 + (int)threadIdx.x;
        const int y = t < g.tokens ? target_of(g, t) : -1;
        const unsigned long long votes = __builtin_amdgcn_ballot_w64(y >= 0);
        if (lane == 0) wave_sum[wave] = __popcll(votes);
        __syncthreads();
        int before = done, all = done;
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        const int c = before + __popcll(votes & ((1ull << lane) - 1));
        if (t < g.tokens) note_row(g, t, y, c);
        done = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) *g.count = done;
}

// The tokens in the order of the group of 128 vocabulary rows that their label
// is in, and within a group in their own order: one workgroup a group (the last
// one only says where the list ends), which counts the labels below its group
// and then puts its own behind them.
__global__ void __launch_bounds__(256)
bucket_kernel(const int *__restrict__ count, const int *__restrict__ label, int2 *member, int *rank, int *bucket)
{
    __shared__ int wave_sum[4];
    const int live = *count, mine = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int below = 0, here = 0;
    for (int c = threadIdx.x; c < live; c += 256) {
        const int b = label[c] / 128;
        below += b < mine;
        here += b == mine;
    }
    for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d);
    if (lane == 0) wave_sum[wave] = below;
    const int any = __syncthreads_or(here);
    int at = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    if (threadIdx.x == 0) bucket[mine] = at;
    if (!any) return;
    for (int c0 = 0; c0 < live; c0 += 256) {
        const int c = c0 + threadIdx.x;
        const bool is = c < live && label[c] / 128 == mine;
        const unsigned long long votes = __builtin_amdgcn_ballot_w64(is);
        __syncthreads();
        if (lane == 0) wave_sum[wave] = __popcll(votes);
        __syncthreads();
        int before = at;
        for (int w = 0; w < 4; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            at += wave_sum[w];
        }
        if (is) {
            const int place = before + __popcll(votes & ((1ull << lane) - 1));
            member[place] = make_int2(c, label[c]);
            rank[c] = place;
        }
    }
}

// One row into its place, padded with zeros to `width` elements, by a workgroup.
template <typename T>
__device__ __forceinline__ void copy_row(const T *__restrict__ from, int cols, T *__restrict__ to, int64_t width)
{
    using V = typename AnyVector<T>::V;
    constexpr int N = 16 / sizeof(T);
    for (int64_t i = threadIdx.x * N; i < width; i += 256 * N) {
        if (i + N <= cols) {
            *reinterpret_cast<vint4 *>(to + i) = *reinterpret_cast<const V *>(from + i);
        } else {
            for (int e = 0; e < N; ++e) to[i + e] = i + e < cols ? from[i + e] : T(0);
        }
    }
}

// dst[c] <- src[rows ? rows[c] : c].  One workgroup a row.
template <typename T>
__global__ void __launch_bounds__(256)
gather_kernel(const T *__restrict__ src, int64_t ld, int cols, const int *rows, const int *count, T *__restrict__ dst,
              int64_t width)
{
    const int c = blockIdx.x;
    if (count && c >= *count) return;
    copy_row<T>(src + (rows ? rows[c] : c) * ld, cols, dst + c * width, width);
}

// Both at once for few rows: a workgroup a row, which finds its place by
// counting the targets before it.
template <typename T>
__global__ void __launch_bounds__(256)
token_gather_kernel(TokenArgs g, const T *__restrict__ src, int64_t ld, int cols, T *__restrict__ dst, int64_t width)
{
    __shared__ int wave_sum[4];
    const int t = blockIdx.x, y = target_of(g, t);
    int before = 0;
    for (int i = threadIdx.x; i < t; i += 256) before += target_of(g, i) >= 0;
    for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = before;
    __syncthreads();
    const int c = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
    if (threadIdx.x == 0) {
        note_row(g, t, y, c);
        if (t == g.tokens - 1) *g.count = c + (y >= 0);
    }
    if (y >= 0) copy_row<T>(src + t * ld, cols, dst + c * width, width);
}

// lse and loss of every compact token from the statistics of the tiles:
// 2^SHIFT tokens a workgroup, the other threads share the tiles.
template <typename T, int SHIFT>
__global__ void __launch_bounds__(256)
loss_kernel(int tiles, const float2 *__restrict__ stats, int64_t ld, const float *__restrict__ target,
            const int *__restrict__ rows, const int *__restrict__ count, float *loss, float *lse)
{
    constexpr int TOKENS = 1 << SHIFT, SLICES = 256 >> SHIFT;
    __shared__ float2 part[SLICES][TOKENS];
    const int live = *count;
    if ((int)blockIdx.x * TOKENS >= live) return;
    const int token = threadIdx.x & (TOKENS - 1), slice = threadIdx.x >> SHIFT;
    const int c = blockIdx.x * TOKENS + token;
    float top = -INFINITY, sum = 0.0f;
    if (c < live) {
        for (int i0 = slice; i0 < tiles; i0 += 4 * SLICES) {
            float2 s[4];
            float t = top;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                s[u] = i0 + SLICES * u < tiles ? stats[(i0 + SLICES * u) * ld + c] : make_float2(-INFINITY, 0.0f);
                t = fmaxf(t, s[u].x);
            }
            const float from = t == -INFINITY ? 0.0f : t;
            // an empty side has sum 0 and maximum -inf: exp(-inf) times 0
            sum *= expf(top - from);
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += s[u].y * expf(s[u].x - from);
            top = t;
        }
    }
    part[slice][token] = make_float2(top, sum);
    for (int half = SLICES / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (slice < half) {
            const float2 a = part[slice][token], b = part[slice + half][token];
            const float t = fmaxf(a.x, b.x), from = t == -INFINITY ? 0.0f : t;
            part[slice][token] = make_float2(t, a.y * expf(a.x - from) + b.y * expf(b.x - from));
        }
    }
    if (slice == 0 && c < live) {
        const float2 a = part[0][token];
        const float l = (a.x == -INFINITY ? 0.0f : a.x) + logf(a.y);
        const int t = rows[c];
        lse[t] = l;
        loss[t] = l - target[c];
    }
}

// gX of every row: the sum over the splits in order (bf16: and what rounding
// took from P at the label), or zeros.  Four elements a thread.
template <typename T>
__global__ void __launch_bounds__(256)
gx_kernel(int hidden, const int *__restrict__ place, const float *__restrict__ part, int64_t ld, int64_t stride,
          int splits, const float *__restrict__ delta, const int *__restrict__ rank, const int *__restrict__ label,
          const T *__restrict__ W, int64_t ldw, T *gx, int64_t ldgx)
{
    const int t = blockIdx.x, c = place[t], h = (int)(blockIdx.y * 256 + threadIdx.x) * 4;
    if (h >= hidden) return;
    const int n = hidden - h < 4 ? hidden - h : 4;
    vfloat4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c >= 0) {
        if (sizeof(T) == 2) {
            const float d = delta[rank[c]];
            const T *w = W + label[c] * ldw + h;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = e < n ? d * to_float(w[e]) : 0.0f;
        }
        const float *p = part + c * ld + h;
        int s = 0;
        for (; s + 4 <= splits; s += 4) {
            vfloat4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const vfloat4 *>(p + (s + u) * stride);
#pragma unroll
            for (int u = 0; u < 4; ++u) v += x[u];
        }
        for (; s < splits; ++s) v += *reinterpret_cast<const vfloat4 *>(p + s * stride);
    }
    T *to = gx + t * ldgx + h;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < n) to[e] = from_float<T>(v[e]);
}

// ---------------------------------------------------------------------------
// sizes
// ---------------------------------------------------------------------------

constexpr int kMaxHidden = 1 << 20, kMaxRows = 1 << 28;

// testing: at most this many vocabulary rows in a piece (0: by size)
std::atomic<int> g_piece_rows{0};

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

bool sizes_ok(int hidden, int tokens, int vocab)
{
    return hidden >= 1 && hidden <= kMaxHidden && tokens >= 0 && tokens <= kMaxRows && vocab >= 1 && vocab <= kMaxRows;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T, Mode MODE, int BM, int BN, int WM, int WN, bool ANY = false>
int launch_tile(const ProductArgs &g, hipStream_t stream)
{
    auto kernel = product_kernel<T, MODE, BM, BN, WM, WN, ANY>;
    constexpr int lds = Product<T, MODE, BM, BN, WM, WN, ANY>::kLds;
    // LDS above the 64 KiB default needs an explicit opt-in, once per kernel and device.
    static std::atomic<unsigned> ready{0};
    int dev = 0;
    HIP_TRY(hipGetDevice(&dev));
    if (dev >= 32 || !(ready.load() >> dev & 1)) {
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    lds));
        if (dev < 32) ready.fetch_or(1u << dev);
    }
    const int64_t tiles = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    if (tiles > 0x7fffffff) {
        g_last_error = "too many tiles for one launch";
        return ULMBLAS_GPU_BAD_ARGUMENT;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, MODE == GX ? (unsigned)g.splits : 1u), dim3(WM * WN * 64), lds,
                       stream, g);
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

// The tile a product of M x N runs on.  N counts tokens in all products but GW.
//  - up to 32 tokens: 128 x 32, of which four workgroups share a CU: the product is bound by the bytes of W then, which
//    may lie on any element (through registers) or on words (straight into LDS);
//  - 256 x 256 where that fills most of the GPU's 256 CUs, with `splits` of k in GX;
//  - else 128 x 128.
enum Tile { NARROW, SMALL, LARGE };
constexpr int kNarrow = 32;
#ifndef SHORT_T
#define SHORT_T 512
#endif
constexpr int kShortTokens = SHORT_T;
template <Mode MODE> Tile tile_for(int M, int N, int tokens, int splits)
{
    if (MODE != GW && N <= kNarrow) return NARROW;
    if (MODE == GW && tokens <= kShortTokens) return SMALL;
    return (int64_t)((M + 255) / 256) * ((N + 255) / 256) * splits >= 200 ? LARGE : SMALL;
}
int tile_rows(Tile t) { return t == LARGE ? 256 : 128; }

// Into how many parts k of GX is cut: two rounds of workgroups if every token
// has a target, as much as it takes with the small tile if there are few tiles.
int splits_of_gx(int hidden, int tokens, int piece)
{
    const int64_t large = ((hidden + 255) / 256) * (int64_t)((tokens + 255) / 256);
    const int64_t small = ((hidden + 127) / 128) * (int64_t)((tokens + 127) / 128);
    const int64_t want = large >= 16 ? 512 / large : 512 / small;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 64), piece / 512));
}

// What the workspace holds and where; every part starts on 256 bytes.
struct Layout {
    int64_t tokens_p, hidden_p;         // rounded up: rows of compact copies, elements of their rows
    int piece;                          // vocabulary rows at a time (gradient: of P; packing: of W)
    int splits;                         // partial sums of gX
    int64_t rows, label, place, lse, both, gloss, delta, target, bucket, member, rank, count, x, w, stats, p, part, bytes;
};

constexpr int64_t kPieceBytes = (int64_t)1 << 30;       // of P or of a packed copy of W, at the most

template <typename T> Layout layout(int hidden, int tokens, int vocab, bool grad)
{
    Layout l{};
    l.tokens_p = round_up(std::max(tokens, 1), 256);
    l.hidden_p = round_up(hidden, kStep<T>);
    const int64_t row = std::max(grad ? l.tokens_p : 0, l.hidden_p) * (int64_t)sizeof(T);
    int64_t piece = std::max<int64_t>(kPieceBytes / row / 256 * 256, 256);
    piece = std::min<int64_t>(piece, 1 << 19);
    if (g_piece_rows.load() > 0) piece = std::min<int64_t>(piece, round_up(g_piece_rows.load(), 256));
    l.piece = (int)std::min<int64_t>(piece, round_up(vocab, 256));
    l.splits = 1;
    if (grad) {
        l.splits = splits_of_gx(hidden, std::max(tokens, 1), l.piece);
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    l.count = take(4);
    l.rows = take(4 * l.tokens_p);
    l.label = take(4 * l.tokens_p);
    l.target = take(4 * l.tokens_p);
    if (grad) {
        l.place = take(4 * l.tokens_p);
        l.lse = take(4 * l.tokens_p);
        l.both = take(4 * l.tokens_p);
        l.gloss = take(4 * l.tokens_p);
        l.delta = take(4 * l.tokens_p);
        l.member = take(8 * l.tokens_p);
        l.rank = take(4 * l.tokens_p);
        l.bucket = take(4 * (round_up(vocab, 128) / 128 + 1));
    }
    l.x = take(l.tokens_p * l.hidden_p * (int64_t)sizeof(T));
    l.w = take((int64_t)l.piece * l.hidden_p * (int64_t)sizeof(T));
    if (!grad) {
        l.stats = take((round_up(vocab, 256) / 128) * l.tokens_p * 8);
    } else {
        l.p = take(l.tokens_p * l.piece * (int64_t)sizeof(T));
        l.part = take((int64_t)l.splits * l.tokens_p * l.hidden_p * 4);
    }
    l.bytes = at;
    return l;
}

template <typename T, Mode MODE> int launch_product(const ProductArgs &g, bool words, hipStream_t stream)
{
    switch (tile_for<MODE>(g.M, g.N, MODE == GW ? g.K : g.N, MODE == GX ? g.splits : 1)) {
    case LARGE: return launch_tile<T, MODE, 256, 256, 2, 4>(g, stream);
    case SMALL: return launch_tile<T, MODE, 128, 128, 2, 2>(g, stream);
    default:
        if constexpr (MODE != GW) {
            if constexpr (sizeof(T) == 2)
                if (!words) return launch_tile<T, MODE, 128, 32, 4, 1, true>(g, stream);
            return launch_tile<T, MODE, 128, 32, 4, 1>(g, stream);
        }
        return ULMBLAS_GPU_BAD_ARGUMENT;        // GW has no narrow tile
    }
}

// Whether W's rows start on 4 bytes, as the copies straight into LDS need them, and whether the product kernel can read
// W where it lies: then, or with the tile for few tokens; a tile's rows are within 31 bits of each other.
template <typename T> bool on_words(const T *W, int ldW) { return ((uintptr_t)W & 3) == 0 && ldW * sizeof(T) % 4 == 0; }
template <typename T> bool in_place(const T *W, int ldW, int tokens)
{
    return (on_words(W, ldW) || tokens <= kNarrow) && (int64_t)ldW * (int64_t)sizeof(T) < (1 << 23);
}

template <typename T>
int gather(const T *src, int64_t ld, int cols, const int *rows, const int *count, int n, T *dst, int64_t width,
           hipStream_t stream)
{
    hipLaunchKernelGGL(gather_kernel<T>, dim3((unsigned)n), dim3(256), 0, stream, src, ld, cols, rows, count, dst,
                       width);
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

// Which tokens count, and their rows of X side by side.
constexpr int kFewTokens = 2048;        // up to here every workgroup counts for itself (a launch less: 4 us)
template <typename T>
int gather_tokens(const TokenArgs &t, const T *X, int64_t ldX, int hidden, T *Xc, int64_t width, hipStream_t stream)
{
    if (t.tokens > 0 && t.tokens <= kFewTokens) {
        hipLaunchKernelGGL(token_gather_kernel<T>, dim3((unsigned)t.tokens), dim3(256), 0, stream, t, X, ldX, hidden, Xc,
                           width);
        HIP_TRY(hipGetLastError());
        return ULMBLAS_GPU_OK;
    }
    hipLaunchKernelGGL(token_kernel, dim3(1), dim3(1024), 0, stream, t);
    HIP_TRY(hipGetLastError());
    return t.tokens > 0 ? gather<T>(X, ldX, hidden, t.rows, t.count, t.tokens, Xc, width, stream) : ULMBLAS_GPU_OK;
}

int bad(const char *text)
{
    g_last_error = text;
    return ULMBLAS_GPU_BAD_ARGUMENT;
}

template <typename T> T *part_of(void *work, int64_t at) { return reinterpret_cast<T *>(static_cast<char *>(work) + at); }

template <typename T>
int xent_device(int hidden, int tokens, int vocab, float alpha, const T *W, int ldW, const T *X, int ldX,
                const int *label, int ignore, float *loss, float *lse, void *work, hipStream_t stream)
{
    if (!sizes_ok(hidden, tokens, vocab)) return bad("invalid size");
    if (ldW < hidden || ldX < hidden) return bad("leading dimension smaller than hidden");
    if (tokens == 0) return ULMBLAS_GPU_OK;
    if (!W || !X || !label || !loss || !lse || !work) return bad("null operand or workspace");
    if ((uintptr_t)work & 15) return bad("workspace not on 16 bytes");
    const Layout l = layout<T>(hidden, tokens, vocab, false);
    TokenArgs t{};
    t.tokens = tokens;
    t.vocab = vocab;
    t.ignore = ignore;
    t.label = label;
    t.loss = loss;
    t.lse_out = lse;
    t.count = part_of<int>(work, l.count);
    t.rows = part_of<int>(work, l.rows);
    t.label_c = part_of<int>(work, l.label);
    T *Xc = part_of<T>(work, l.x);
    int rc = gather_tokens<T>(t, X, ldX, hidden, Xc, l.hidden_p, stream);
    if (rc) return rc;

    ProductArgs g{};
    g.B = Xc;
    g.ldB = l.hidden_p * (int64_t)sizeof(T);
    g.widthB = (int)l.hidden_p;
    g.N = tokens;
    g.K = hidden;
    g.count = t.count;
    g.alpha = alpha;
    g.label = t.label_c;
    g.ldStats = l.tokens_p;
    g.target = part_of<float>(work, l.target);
    const bool direct = in_place(W, ldW, tokens), words = !direct || on_words(W, ldW);
    const int piece = direct ? vocab : l.piece;
    int tiles = 0;
    for (int v0 = 0; v0 < vocab; v0 += piece) {
        g.M = std::min(piece, vocab - v0);
        g.first = v0;
        if (direct) {
            g.A = W;
            g.ldA = (int64_t)ldW * sizeof(T);
            g.widthA = hidden;
        } else {
            T *Wp = part_of<T>(work, l.w);
            if ((rc = gather<T>(W + (int64_t)v0 * ldW, ldW, hidden, nullptr, nullptr, g.M, Wp, l.hidden_p, stream)))
                return rc;
            g.A = Wp;
            g.ldA = l.hidden_p * (int64_t)sizeof(T);
            g.widthA = (int)l.hidden_p;
        }
        g.stats = part_of<float2>(work, l.stats) + (int64_t)tiles * l.tokens_p;
        if ((rc = launch_product<T, STATS>(g, words, stream))) return rc;
        const int bm = tile_rows(tile_for<STATS>(g.M, g.N, g.N, 1));
        tiles += (g.M + bm - 1) / bm;
    }
    if (tokens <= 256) {
        hipLaunchKernelGGL((loss_kernel<T, 0>), dim3((unsigned)tokens), dim3(256), 0, stream, tiles,
                           part_of<float2>(work, l.stats), l.tokens_p, g.target, t.rows, t.count, loss, lse);
    } else {
        hipLaunchKernelGGL((loss_kernel<T, 4>), dim3((unsigned)((tokens + 15) / 16)), dim3(256), 0, stream, tiles,
                           part_of<float2>(work, l.stats), l.tokens_p, g.target, t.rows, t.count, loss, lse);
    }
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

template <typename T>
int xent_grad_device(int hidden, int tokens, int vocab, float alpha, const T *W, int ldW, const T *X, int ldX,
                     const int *label, int ignore, const float *lse, const float *gloss, const float *glse, float beta,
                     T *gW, int ldGW, T *gX, int ldGX, void *work, hipStream_t stream)
{
    if (!sizes_ok(hidden, tokens, vocab)) return bad("invalid size");
    if (ldW < hidden || ldX < hidden || (gW && ldGW < hidden) || (gX && ldGX < hidden))
        return bad("leading dimension smaller than hidden");
    if (!gW && !gX) return ULMBLAS_GPU_OK;
    if (tokens > 0 && (!W || !X || !label || !lse || !gloss)) return bad("null operand");
    if (!work) return bad("null workspace");
    if ((uintptr_t)work & 15) return bad("workspace not on 16 bytes");
    const Layout l = layout<T>(hidden, tokens, vocab, true);
    TokenArgs t{};
    t.tokens = tokens;
    t.vocab = vocab;
    t.ignore = ignore;
    t.label = label;
    t.count = part_of<int>(work, l.count);
    t.rows = part_of<int>(work, l.rows);
    t.label_c = part_of<int>(work, l.label);
    t.place = part_of<int>(work, l.place);
    t.lse = lse;
    t.gloss = gloss;
    t.glse = glse;
    t.alpha = alpha;
    t.lse_c = part_of<float>(work, l.lse);
    t.both_c = part_of<float>(work, l.both);
    t.gloss_c = part_of<float>(work, l.gloss);
    T *Xc = part_of<T>(work, l.x), *P = part_of<T>(work, l.p);
    int rc = gather_tokens<T>(t, X, ldX, hidden, Xc, l.hidden_p, stream);
    if (rc) return rc;
    float *delta = part_of<float>(work, l.delta);
    int2 *member = part_of<int2>(work, l.member);
    int *rank = part_of<int>(work, l.rank), *bucket = part_of<int>(work, l.bucket);
    if (sizeof(T) == 2) {
        hipLaunchKernelGGL(bucket_kernel, dim3((unsigned)(round_up(vocab, 128) / 128 + 1)), dim3(256), 0, stream, t.count,
                           t.label_c, member, rank, bucket);
        HIP_TRY(hipGetLastError());
    }
    // P: rows of blocks; all of them
    const int64_t row_x = l.hidden_p * (int64_t)sizeof(T), row_p = (int64_t)l.piece / kStep<T> * kBlockBytes;
    const int blocks_p = (int)(l.tokens_p / kBlockTokens * (l.piece / kStep<T>));
    const bool direct = in_place(W, ldW, tokens), words = !direct || on_words(W, ldW);
    for (int v0 = 0; v0 < vocab; v0 += l.piece) {
        const int vn = std::min(l.piece, vocab - v0);
        const T *Wv = W ? W + (int64_t)v0 * ldW : nullptr;
        int64_t row_w = (int64_t)ldW * (int64_t)sizeof(T);
        int width_w = hidden;
        ProductArgs g{};
        g.count = t.count;
        g.alpha = alpha;
        if (tokens > 0) {
            if (!direct) {
                T *Wp = part_of<T>(work, l.w);
                if ((rc = gather<T>(Wv, ldW, hidden, nullptr, nullptr, vn, Wp, l.hidden_p, stream))) return rc;
                Wv = Wp;
                row_w = row_x;
                width_w = (int)l.hidden_p;
            }
            g.A = Wv;
            g.ldA = row_w;
            g.widthA = width_w;
            g.B = Xc;
            g.ldB = row_x;
            g.widthB = (int)l.hidden_p;
            g.M = vn;
            g.N = tokens;
            g.K = hidden;
            g.label = t.label_c;
            g.first = v0;
            g.lse = t.lse_c;
            g.both = t.both_c;
            g.gloss = t.gloss_c;
            g.P = P;
            g.ldP = row_p;
            g.rank = rank;
            g.delta = delta;
            if ((rc = launch_product<T, PROB>(g, words, stream))) return rc;
        }
        if (gX && tokens > 0) {
            g.A = Wv;
            g.ldA = row_w;
            g.widthA = width_w;
            g.B = P;
            g.ldB = row_p;
            g.widthB = blocks_p;
            g.M = hidden;
            g.N = tokens;
            g.K = vn;
            g.part = part_of<float>(work, l.part);
            g.ldD = l.hidden_p;
            g.splitStride = l.tokens_p * l.hidden_p;
            g.splits = l.splits;
            g.add = v0 > 0;
            if ((rc = launch_product<T, GX>(g, words, stream))) return rc;
        }
        if (gW) {
            g.A = Xc;
            g.ldA = row_x;
            g.widthA = (int)l.hidden_p;
            g.B = P;
            g.ldB = row_p;
            g.widthB = blocks_p;
            g.M = hidden;
            g.N = vn;
            g.K = tokens;
            g.first = v0;
            g.delta = delta;
            g.bucket = bucket;
            g.member = member;
            g.out = gW + (int64_t)v0 * ldGW;
            g.ldD = ldGW;
            g.beta = beta;
            if ((rc = launch_product<T, GW>(g, words, stream))) return rc;
        }
    }
    if (gX && tokens > 0) {
        hipLaunchKernelGGL(gx_kernel<T>, dim3((unsigned)tokens, (unsigned)((hidden + 1023) / 1024)), dim3(256), 0, stream, hidden, t.place,
                           part_of<float>(work, l.part), l.hidden_p, l.tokens_p * l.hidden_p, l.splits, delta, rank,
                           t.label_c, W, (int64_t)ldW, gX,
                           (int64_t)ldGX);
        HIP_TRY(hipGetLastError());
    }
    return ULMBLAS_GPU_OK;
}

template <typename T> long worksize(int hidden, int tokens, int vocab, bool grad)
{
    if (!sizes_ok(hidden, tokens, vocab)) return 0;
    return (long)layout<T>(hidden, tokens, vocab, grad).bytes;
}

}  // namespace

void xent_set_piece_rows(int rows) { g_piece_rows.store(rows); }

}  // namespace ulmgpu

extern "C" {

long ulmblas_gpu_sxent_worksize(int hidden, int tokens, int vocab) { return worksize<float>(hidden, tokens, vocab, false); }
long ulmblas_gpu_bxent_worksize(int hidden, int tokens, int vocab) { return worksize<bf16_t>(hidden, tokens, vocab, false); }
long ulmblas_gpu_sxent_grad_worksize(int hidden, int tokens, int vocab)
{
    return worksize<float>(hidden, tokens, vocab, true);
}
long ulmblas_gpu_bxent_grad_worksize(int hidden, int tokens, int vocab)
{
    return worksize<bf16_t>(hidden, tokens, vocab, true);
}

int ulmblas_gpu_sxent(int hidden, int tokens, int vocab, float alpha, const float *dW, int ldW, const float *dX, int ldX,
                      const int *dLabel, int ignore, float *dLoss, float *dLse, void *work, void *stream)
{
    return xent_device<float>(hidden, tokens, vocab, alpha, dW, ldW, dX, ldX, dLabel, ignore, dLoss, dLse, work,
                              static_cast<hipStream_t>(stream));
}

int ulmblas_gpu_bxent(int hidden, int tokens, int vocab, float alpha, const unsigned short *dW, int ldW,
                      const unsigned short *dX, int ldX, const int *dLabel, int ignore, float *dLoss, float *dLse,
                      void *work, void *stream)
{
    return xent_device<bf16_t>(hidden, tokens, vocab, alpha, dW, ldW, dX, ldX, dLabel, ignore, dLoss, dLse, work,
                               static_cast<hipStream_t>(stream));
}

int ulmblas_gpu_sxent_grad(int hidden, int tokens, int vocab, float alpha, const float *dW, int ldW, const float *dX,
                           int ldX, const int *dLabel, int ignore, const float *dLse, const float *dGLoss,
                           const float *dGLse, float beta, float *dGW, int ldGW, float *dGX, int ldGX, void *work,
                           void *stream)
{
    return xent_grad_device<float>(hidden, tokens, vocab, alpha, dW, ldW, dX, ldX, dLabel, ignore, dLse, dGLoss, dGLse,
                                   beta, dGW, ldGW, dGX, ldGX, work, static_cast<hipStream_t>(stream));
}

int ulmblas_gpu_bxent_grad(int hidden, int tokens, int vocab, float alpha, const unsigned short *dW, int ldW,
                           const unsigned short *dX, int ldX, const int *dLabel, int ignore, const float *dLse,
                           const float *dGLoss, const float *dGLse, float beta, unsigned short *dGW, int ldGW,
                           unsigned short *dGX, int ldGX, void *work, void *stream)
{
    return xent_grad_device<bf16_t>(hidden, tokens, vocab, alpha, dW, ldW, dX, ldX, dLabel, ignore, dLse, dGLoss, dGLse,
                                    beta, dGW, ldGW, dGX, ldGX, work, static_cast<hipStream_t>(stream));
}

}  // extern "C"
