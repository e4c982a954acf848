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
#include <initializer_list>
#include <utility>

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
gx_kernel(int hidden, const int *__restrict__ place, const int *__restrict__ count, int rows, int columns, int groups,
          int steps, const float *__restrict__ part, int64_t ld, const float *__restrict__ delta, const int *__restrict__ rank, const int *__restrict__ label,
          const T *__restrict__ W, int64_t ldw, T *gx, int64_t ldgx)
{
    const int t = blockIdx.x, c = place[t], h = (int)(blockIdx.y * 256 + threadIdx.x) * 4;
    const int live = *count, tiles = (hidden + rows - 1) / rows * ((live + columns - 1) / columns);
    const int splits = splits_of(groups, tiles, steps, live, hidden);
    if (h >= hidden) return;
    const int n = hidden - h < 4 ? hidden - h : 4;
    vfloat4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c >= 0) {
        if (sizeof(T) == 2) {
            const float d = delta[rank ? rank[c] : c];
            const T *w = W + label[c] * ldw + h;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = e < n ? d * to_float(w[e]) : 0.0f;
        }
        const int64_t stride = live * ld;
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

// A launch has fewer than 2^32 threads, and some have a workgroup of 256 for each token.
constexpr int kMaxHidden = 1 << 20, kMaxTokens = 1 << 23, kMaxVocab = 1 << 28, kMaxLd = (1 << 21) - 1;

// testing: at most this many vocabulary rows in a piece (0: by size)
std::atomic<int> g_piece_rows{0};

inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

bool sizes_ok(int hidden, int tokens, int vocab)
{
    return hidden >= 1 && hidden <= kMaxHidden && tokens >= 0 && tokens <= kMaxTokens && vocab >= 1 && vocab <= kMaxVocab;
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

template <typename T, Mode MODE, int BM, int BN, int WM, int WN, int BUFFERS = 2, bool ANY = false>
int launch_tile(const ProductArgs &g, hipStream_t stream)
{
    auto kernel = product_kernel<T, MODE, BM, BN, WM, WN, BUFFERS, ANY>;
    constexpr int lds = Product<T, MODE, BM, BN, WM, WN, BUFFERS, ANY>::kLds;
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
    if (std::max<int64_t>(tiles, g.groups) * WM * WN * 64 >> 32) {
        g_last_error = "too many tiles for one launch";
        return ULMBLAS_GPU_BAD_ARGUMENT;
    }
    // a single step of k needs one tile of LDS, and what the result is staged in
    constexpr int one = std::max(Product<T, MODE, BM, BN, WM, WN, BUFFERS, ANY>::kStage, BM * BN * 2);
    const bool single = BUFFERS == 2 && !ANY && MODE == GW && g.K <= kStep<T>;
    const unsigned grid = (unsigned)(MODE == GX ? std::max<int64_t>(tiles, g.groups) : tiles);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(WM * WN * 64), single ? one : lds, stream, g);
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

// The tile a product runs on: the one with the least estimated time.  The CUs
// share the tiles, so the CU with the most of them counts:
//
//   time = ceil(tiles / 256) * (rows * columns * K / (rate * efficiency) + overhead)
//
// in microseconds, with the rate of the 256 x 256 tile on large products (bf16
// 1250 TFLOP/s, fp32 122) and what the others reached on the same ones (tokens
// 2048, hidden 1024; bf16 vocabulary 32768, fp32 16384):
//
//                 logits                GX                 overhead (beginning, end; writing for GW)
//   256 x 256     127 us / 566 us       145 us / 562 us    8.5   12
//   128 x 128     151    / 595          135    / 574       1.5    3.2 (2.2 with a single step of k)
//   128 x 64      184    / 605          181    / 596       1.5
//   128 x 32             / 666                 / 650       1.5
//
// (bf16 tiles other than the largest lose more with a longer k: 512 tokens, hidden 4096: 150 us against 120.)
// How many of the tokens count is not known here: all of them decide for three
// parts, three quarters and half of them for one part each.  The tile for 32
// columns is bf16's up to 32 tokens (wider products would write P past its rows
// with it); where W lies off words the logits take it with half its rows (through
// registers: twice the workgroups keep as many bytes on the way; one token
// against 1410 x 6230: 92 -> 73 us).  GX may cut k, so that any tile fills the
// GPU: it counts fractions of rounds.
struct Tile {
    int rows, columns;
};
constexpr Tile kTiles[] = {{256, 256}, {128, 128}, {128, 64}, {128, 32}}, kAnyTile = {64, 32};
constexpr int kNarrow = 32;
constexpr int kGroups = 512;            // workgroups GX is spread over: two rounds, so that some tokens may be missing

template <typename T, Mode MODE> Tile choose(int M, int N, int K, bool words = true)
{
    constexpr bool half = sizeof(T) == 2;
    if (half && MODE != GW && N <= kNarrow) return words || MODE == GX ? kTiles[3] : kAnyTile;
    constexpr double rate = half ? 2.44e6 : 0.238e6;            // products and sums a CU and microsecond
    constexpr double efficiency[4] = {1.0, half ? 0.75 : 0.95, half ? 0.65 : 0.93, 0.84};
    int best = 0;
    double least = 0.0;
    for (int t = 0; t < 4; ++t) {
        if ((MODE == GW && t > 1) || (half && t == 3)) continue;
        double time = 0.0;
        for (int quarters = 2; quarters <= 4; ++quarters) {
            const int n = MODE == GW ? N : std::max(1, (int)((int64_t)N * quarters / 4));
            const int kk = MODE == GW ? std::max(1, (int)((int64_t)K * quarters / 4)) : K;
            const double tiles = (double)((M + kTiles[t].rows - 1) / kTiles[t].rows) *
                                 ((n + kTiles[t].columns - 1) / kTiles[t].columns);
            const double rounds = MODE == GX ? std::max(1.0, tiles / 256) : std::ceil(tiles / 256);
            double k = kk, overhead = t == 0 ? 8.5 : 1.5;
            if (MODE == GX) k = k * std::min(1.0, std::max(tiles / 256, 8.0 * kStep<T> / kk));
            if (MODE == GW) overhead = t == 0 ? 12.0 : K <= kStep<T> ? 2.2 : 3.2;
            time += (quarters == 4 ? 3 : 1) * rounds * (kTiles[t].rows * kTiles[t].columns * k / (rate * efficiency[t]) + overhead);
        }
        if (t == 0 || time < least) {
            best = t;
            least = time;
        }
    }
    return kTiles[best];
}

template <typename T, Mode MODE> int launch_product(const ProductArgs &g, Tile tile, bool words, hipStream_t stream)
{
    const int64_t groups = (int64_t)((g.M + tile.rows - 1) / tile.rows) * ((g.N + tile.columns - 1) / tile.columns);
    if (tile.rows == 256) return launch_tile<T, MODE, 256, 256, 2, 4>(g, stream);
    if constexpr (MODE == GW) {
        return launch_tile<T, MODE, 128, 128, 2, 2>(g, stream);
    } else {
        if (tile.columns == 32) {
            if constexpr (sizeof(T) == 2)
                if (!words) return launch_tile<T, MODE, MODE == GX ? 128 : 64, 32, 4, 1, 2, true>(g, stream);
            return launch_tile<T, MODE, 128, 32, 4, 1, 4>(g, stream);
        }
        if (tile.columns == 64) return launch_tile<T, MODE, 128, 64, 2, 2, 3>(g, stream);
        // alone on its CU a workgroup keeps more steps open
        if (MODE != GX && groups <= 256) return launch_tile<T, MODE, 128, 128, 2, 2, 4>(g, stream);
        return launch_tile<T, MODE, 128, 128, 2, 2>(g, stream);
    }
}

// What the workspace holds and where; every part starts on 256 bytes.
struct Layout {
    int64_t tokens_p, hidden_p;         // rounded up: rows of compact copies, elements of their rows
    int piece;                          // vocabulary rows at a time (gradient: of P; packing: of W)
    int64_t rows, label, place, lse, both, gloss, delta, target, bucket, member, rank, count, x, w, stats, p, part, bytes;
};

// of P and of a packed copy of W in the gradient, and of a packed copy of W in the forward call, at the most (where 256
// rows are not more)
constexpr int64_t kPieceBytes = (int64_t)1 << 30, kPackBytes = (int64_t)1 << 27;

template <typename T> Layout layout(int hidden, int tokens, int vocab, bool grad)
{
    Layout l{};
    l.tokens_p = round_up(std::max(tokens, 1), 256);
    l.hidden_p = round_up(hidden, kStep<T>);
    // bf16 may have to pack its piece of W; a piece is at most 2^19 rows, and all are about as long
    const bool packs = sizeof(T) == 2 && tokens > kNarrow;
    const int64_t row = std::max(grad ? l.tokens_p : 1, packs ? l.hidden_p : 1) * (int64_t)sizeof(T);
    int64_t most = std::min<int64_t>(std::max<int64_t>((grad ? kPieceBytes : kPackBytes) / row / 256 * 256, 256), 1 << 19);
    if (g_piece_rows.load() > 0) most = std::min<int64_t>(most, round_up(g_piece_rows.load(), 256));
    const int64_t pieces = (vocab + most - 1) / most;
    l.piece = (int)round_up((vocab + pieces - 1) / pieces, 256);
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
    l.w = take(packs ? (int64_t)l.piece * l.hidden_p * (int64_t)sizeof(T) : 0);
    if (!grad) {
        // a tile has 128 rows at least, but for few tokens of bf16, whose W may lie off words
        const int rows = sizeof(T) == 2 && tokens <= kNarrow ? kAnyTile.rows : kTiles[1].rows;
        l.stats = take((round_up(vocab, 256) / rows) * l.tokens_p * 8);
    } else {
        l.p = take(l.tokens_p * l.piece * (int64_t)sizeof(T));
        // as many splits as fill kGroups workgroups with tiles, or one
        const Tile gx = choose<T, GX>(hidden, std::max(tokens, 1), l.piece);
        l.part = take(std::max((int64_t)kGroups * gx.rows * gx.columns, l.tokens_p * l.hidden_p) * 4);
    }
    l.bytes = at;
    return l;
}

// Whether W's rows start on 4 bytes, as the copies straight into LDS need them, and whether the product kernel can read
// W where it lies: then, or with the tile for few tokens.
template <typename T> bool on_words(const T *W, int ldW) { return ((uintptr_t)W & 3) == 0 && ldW * sizeof(T) % 4 == 0; }
template <typename T> bool in_place(const T *W, int ldW, int tokens)
{
    return on_words(W, ldW) || tokens <= kNarrow;
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

template <typename T> bool off(const void *p) { return (uintptr_t)p % sizeof(T) != 0; }

// Memory that a call reads or writes: `columns` runs of `bytes`, `pitch` apart.
struct Window {
    uintptr_t at;
    int64_t bytes, pitch, columns;
    uintptr_t end() const { return at + (uintptr_t)((columns - 1) * pitch + bytes); }
};
template <typename T> Window matrix(const T *p, int rows, int columns, int ld)
{
    return {(uintptr_t)p, rows * (int64_t)sizeof(T), ld * (int64_t)sizeof(T), p ? columns : 0};
}
template <typename T> Window vector(const T *p, int64_t n)
{
    return {(uintptr_t)p, n * (int64_t)sizeof(T), n * (int64_t)sizeof(T), p && n > 0 ? 1 : 0};
}

// Whether two windows share a byte.  One may lie in the gaps between the other's columns (the halves of one wide matrix):
// every column of the one with fewer of them that lies inside the other is compared with the two columns it can meet,
// after a single comparison for all of them where the columns are equally far apart.
bool meet(Window a, Window b)
{
    if (a.columns <= 0 || b.columns <= 0 || a.at >= b.end() || b.at >= a.end()) return false;
    if (a.columns > b.columns) std::swap(a, b);
    auto met = [&](uintptr_t from) {            // by a column of a
        const int64_t k = from <= b.at ? 0 : std::min<int64_t>((int64_t)((from - b.at) / (uintptr_t)b.pitch), b.columns - 1);
        for (int64_t i = k; i < std::min(k + 2, b.columns); ++i) {
            const uintptr_t at = b.at + (uintptr_t)(i * b.pitch);
            if (from < at + (uintptr_t)b.bytes && at < from + (uintptr_t)a.bytes) return true;
        }
        return false;
    };
    // the first column of a that ends behind b's beginning, the last one that begins before b's end
    const int64_t first = a.at + (uintptr_t)a.bytes > b.at
                              ? 0 : (int64_t)((b.at - a.at - (uintptr_t)a.bytes) / (uintptr_t)a.pitch) + 1;
    const int64_t last = std::min(a.columns - 1, (int64_t)((b.end() - 1 - a.at) / (uintptr_t)a.pitch));
    if (a.pitch == b.pitch) {
        // columns between the ends meet what the ones before them met; at the ends a neighbour may be missing
        return first <= last && (met(a.at + (uintptr_t)(first * a.pitch)) || met(a.at + (uintptr_t)(last * a.pitch)));
    }
    for (int64_t i = first; i <= last; ++i)
        if (met(a.at + (uintptr_t)(i * a.pitch))) return true;
    return false;
}

// Whether what a call writes (the first `written` windows) shares memory with anything else it is given.
bool overlapping(std::initializer_list<Window> windows, int written)
{
    const Window *w = windows.begin();
    const int n = (int)windows.size();
    for (int i = 0; i < written; ++i)
        for (int j = i + 1; j < n; ++j)
            if (meet(w[i], w[j])) return true;
    return false;
}

template <typename T> T *part_of(void *work, int64_t at) { return reinterpret_cast<T *>(static_cast<char *>(work) + at); }

template <typename T> long worksize(int hidden, int tokens, int vocab, bool grad)
{
    if (!sizes_ok(hidden, tokens, vocab)) return 0;
    if (grad && xent_takes_few(hidden, tokens)) return xent_few_worksize(hidden, tokens, vocab);
    return (long)layout<T>(hidden, tokens, vocab, grad).bytes;
}

template <typename T>
int xent_device(int hidden, int tokens, int vocab, float alpha, const T *W, int ldW, const T *X, int ldX,
                const int *label, int ignore, float *loss, float *lse, void *work, hipStream_t stream)
{
    if (!sizes_ok(hidden, tokens, vocab)) return bad("invalid size");
    if (ldW < hidden || ldX < hidden) return bad("leading dimension smaller than hidden");
    if (ldW > kMaxLd) return bad("leading dimension of W beyond 2^21");
    if (tokens == 0) return ULMBLAS_GPU_OK;
    if (!W || !X || !label || !loss || !lse || !work) return bad("null operand or workspace");
    if (off<T>(W) || off<T>(X) || off<int>(label) || off<float>(loss) || off<float>(lse))
        return bad("operand off its type's alignment");
    if ((uintptr_t)work & 15) return bad("workspace not on 16 bytes");
    const Layout l = layout<T>(hidden, tokens, vocab, false);
    if (overlapping({vector(loss, tokens), vector(lse, tokens), vector(static_cast<char *>(work), l.bytes),
                     matrix(W, hidden, vocab, ldW), matrix(X, hidden, tokens, ldX), vector(label, tokens)}, 3))
        return bad("a result or the workspace overlaps another operand");
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
    // as many rows at a time as one launch has tiles for (128 x 64 ones, 256 threads each)
    int64_t most = tokens <= kNarrow ? kMaxVocab : ((int64_t)1 << 36) / tokens / 256 * 256;
    if (g_piece_rows.load() > 0) most = std::min<int64_t>(most, round_up(g_piece_rows.load(), 256));
    const int piece = (int)std::min<int64_t>(direct ? vocab : l.piece, most);
    int tiles = 0;
    for (int v0 = 0; v0 < vocab; v0 += piece) {
        g.M = std::min(piece, vocab - v0);
        g.first = v0;
        if (direct) {
            g.A = W + (int64_t)v0 * ldW;
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
        const Tile tile = choose<T, STATS>(g.M, g.N, g.K, words);
        if ((rc = launch_product<T, STATS>(g, tile, words, stream))) return rc;
        tiles += (g.M + tile.rows - 1) / tile.rows;
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
    if (ldW > kMaxLd) return bad("leading dimension of W beyond 2^21");
    if (!gW && !gX) return ULMBLAS_GPU_OK;
    if (tokens > 0 && (!W || !X || !label || !lse || !gloss)) return bad("null operand");
    if (!work) return bad("null workspace");
    if (off<T>(W) || off<T>(X) || off<T>(gW) || off<T>(gX) || off<int>(label) || off<float>(lse) || off<float>(gloss) ||
        off<float>(glse))
        return bad("operand off its type's alignment");
    if ((uintptr_t)work & 15) return bad("workspace not on 16 bytes");
    // without tokens nothing but gW is touched
    if (overlapping({matrix(gW, hidden, vocab, ldGW), matrix(gX, hidden, tokens, ldGX),
                     vector(static_cast<char *>(work), worksize<T>(hidden, tokens, vocab, true)),
                     matrix(W, hidden, tokens ? vocab : 0, ldW), matrix(X, hidden, tokens, ldX), vector(label, tokens),
                     vector(lse, tokens), vector(gloss, tokens), vector(glse, tokens)}, 3))
        return bad("a result or the workspace overlaps another operand");
    if (xent_takes_few(hidden, tokens))
        return xent_few_grad<T>(hidden, tokens, vocab, alpha, W, ldW, X, ldX, label, ignore, lse, gloss, glse, beta, gW, ldGW,
                                gX, ldGX, static_cast<float *>(work), stream);
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
    int *rank = tokens > kUnsorted ? part_of<int>(work, l.rank) : nullptr, *bucket = part_of<int>(work, l.bucket);
    if (sizeof(T) == 2 && tokens > kUnsorted) {
        hipLaunchKernelGGL(bucket_kernel, dim3((unsigned)(round_up(vocab, 128) / 128 + 1)), dim3(256), 0, stream, t.count,
                           t.label_c, member, rank, bucket);
        HIP_TRY(hipGetLastError());
    }
    // P: rows of blocks; all of them
    const int64_t row_x = l.hidden_p * (int64_t)sizeof(T), row_p = (int64_t)l.piece / kStep<T> * kBlockBytes;
    const int blocks_p = (int)(l.tokens_p / kBlockTokens * (l.piece / kStep<T>));
    const bool direct = in_place(W, ldW, tokens), words = !direct || on_words(W, ldW);
    const Tile gx_tile = choose<T, GX>(hidden, std::max(tokens, 1), l.piece);
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
            if ((rc = launch_product<T, PROB>(g, choose<T, PROB>(g.M, g.N, g.K, words), words, stream))) return rc;
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
            g.groups = kGroups;
            g.steps = (l.piece + kStep<T> - 1) / kStep<T>;
            g.add = v0 > 0;
            if ((rc = launch_product<T, GX>(g, gx_tile, words, stream))) return rc;
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
            g.label = t.label_c;
            g.rank = rank;
            g.delta = delta;
            g.bucket = bucket;
            g.member = member;
            g.out = gW + (int64_t)v0 * ldGW;
            g.ldD = ldGW;
            g.beta = beta;
            g.past = (int64_t)vocab * hidden * (int64_t)sizeof(T) > kPastCaches;
            if ((rc = launch_product<T, GW>(g, choose<T, GW>(g.M, g.N, g.K), words, stream))) return rc;
        }
    }
    if (gX && tokens > 0) {
        hipLaunchKernelGGL(gx_kernel<T>, dim3((unsigned)tokens, (unsigned)((hidden + 1023) / 1024)), dim3(256), 0, stream, hidden, t.place,
                           t.count, gx_tile.rows, gx_tile.columns, kGroups, (l.piece + kStep<T> - 1) / kStep<T>,
                           part_of<float>(work, l.part), l.hidden_p, delta, rank,
                           t.label_c, W, (int64_t)ldW, gX,
                           (int64_t)ldGX);
        HIP_TRY(hipGetLastError());
    }
    return ULMBLAS_GPU_OK;
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
