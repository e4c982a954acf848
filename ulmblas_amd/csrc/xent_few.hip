// The gradient of the softmax cross entropy (xent.hip) for up to 8 tokens, in one
// pass over W.
//
// With a handful of tokens the products are inner products, and W is read once
// for all three of them: a workgroup holds ROWS rows of W in registers, 8
// consecutive elements a thread (EIGHTS times 8 for long rows), next to the same
// elements of every token's x and of its part of every token's gX.  The logits of
// the rows come out of one exchange between the lanes (which halves the values
// as it doubles the lanes summed over) and one through LDS between the waves;
// every wave then has all of P in its lanes and takes it as scalars for
//
//     gX_t += P_vt w_v   (registers, written once at the end)
//     gW_v  = sum_t P_vt x_t + beta gW_v   (stored as it is made)
//
// P stays in fp32.  The next rows are on their way while these are worked on.
// Measured (vocabulary 32768, hidden 4096): bf16 1 - 2 tokens 108 us and 4 tokens
// 118 us, which the bytes of W and gW bound (4.5 - 5.0 TB/s), 8 tokens 165 - 175 us, bound by
// the 24 multiplications and additions an element of W and their operands' conversion;
// fp32 205 - 233 us.  The three products as such take 230 and 415 us.  5 x 1001 x 30001
// bf16: 43 us (70 us by the products), 36 of them in this pass, which moves 141 MB, 20 of
// them partial sums of gX (3.9 TB/s).  A kernel for each count of tokens: with values
// for the next power of two computed too, that pass took 46 us.
// The exchange between lanes goes through swaps and DPP: through LDS it was the
// longest part of the work on a set of rows (2 tokens, hidden 1024: 83 -> 34 us).

#include "internal.h"
#include "xent_kernel.hip.h"

#include <algorithm>

using namespace ulmgpu::xent;

namespace ulmgpu {
namespace {

struct FewArgs {
    int hidden, vocab, ignore;
    float alpha, beta;
    const void *W, *X;
    int64_t ldW, ldX, ldGW;
    const int *label;
    const float *lse, *gloss, *glse;
    void *gW;                   // null: not wanted
    float *part;                // [workgroup][token][hidden] (null: gX not wanted)
};

template <typename T> struct Eight {        // 8 consecutive elements as they lie in memory
    static constexpr int WORDS = 2 * (int)sizeof(T);
    unsigned w[WORDS];
    __device__ __forceinline__ float at(int e) const
    {
        if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        else return __uint_as_float(w[e]);
    }
    // elements 0 .. n-1 of p, zeros beyond
    __device__ __forceinline__ void load(const T *p, int n)
    {
        using V = typename AnyVector<T>::V;
        if (n >= 8) {
#pragma unroll
            for (int q = 0; q < WORDS / 4; ++q) {
                const vint4 v = *reinterpret_cast<const V *>(p + q * (16 / sizeof(T)));
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * q + i] = (unsigned)v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (e >= n) continue;
                if constexpr (sizeof(T) == 2) w[e >> 1] |= (unsigned)p[e] << 16 * (e & 1);
                else w[e] = __float_as_uint(p[e]);
            }
        }
    }
};

template <typename T> __device__ __forceinline__ void store_eight(T *p, const float (&x)[8], int n)
{
    using V = typename AnyVector<T>::V;
    if (n >= 8) {
#pragma unroll
        for (int q = 0; q < 8 * (int)sizeof(T) / 16; ++q) {
            vint4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2)
                    v[i] = (int)((unsigned)from_float<T>(x[2 * i]) | (unsigned)from_float<T>(x[2 * i + 1]) << 16);
                else
                    v[i] = __float_as_int(x[4 * q + i]);
            }
            *reinterpret_cast<V *>(p + q * (16 / sizeof(T))) = v;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = from_float<T>(x[e]);
    }
}

// The sum over the two lanes that differ in one bit of their number (32, 16, 8:
// that bit alone; 4: mirrored within 8 lanes; 2, 1), of a where the bit is clear
// and of b where it is set.
template <int MASK> __device__ __forceinline__ float halve(float a, float b, int lane)
{
    if constexpr (MASK == 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    } else if constexpr (MASK == 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    } else {
        constexpr int CTRL = MASK == 8 ? 0x128 : MASK == 4 ? 0x141 : MASK == 2 ? 0x4e : 0xb1;
        const bool upper = (lane & MASK) != 0;
        const float keep = upper ? b : a, send = upper ? a : b;
        return keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(send), CTRL, 0xf, 0xf, false));
    }
}
// z[0] becomes the sum over the wave of z[lane >> (6 - log2 N)]: each step halves the values a lane holds.
template <int N, int MASK = 32> __device__ __forceinline__ void sum_over_wave(float *z, int lane)
{
    if constexpr (MASK >= 1) {
        if constexpr (N > 1) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) z[i] = halve<MASK>(z[i], z[i + N / 2], lane);
            sum_over_wave<N / 2, MASK / 2>(z, lane);
        } else {
            z[0] = halve<MASK>(z[0], z[0], lane);
            sum_over_wave<1, MASK / 2>(z, lane);
        }
    }
}

// TOKENS tokens; values are laid out for the next power of two.
template <typename T, int TOKENS, int EIGHTS, int ROWS>
__global__ void __launch_bounds__(512, 2) few_kernel(FewArgs g)
{
    constexpr int PITCH = TOKENS <= 2 ? TOKENS : TOKENS <= 4 ? 4 : 8;
    constexpr int N = ROWS * PITCH;                 // values a chunk of rows makes: row * PITCH + token
    static_assert(N <= 64 && (N & (N - 1)) == 0, "one value a lane");
    constexpr int LOG = N == 64 ? 6 : N == 32 ? 5 : N == 16 ? 4 : N == 8 ? 3 : N == 4 ? 2 : N == 2 ? 1 : 0;
    __shared__ float sums[2][8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const T *W = static_cast<const T *>(g.W);
    const int pitch = blockDim.x * 8;               // elements from one of a thread's eights to the next

    // this lane's value, and what belongs to its token
    const int mine = lane >> (6 - LOG), my_row = mine / PITCH, my_token = mine % PITCH;
    int want = -1;
    float lse = 0.0f, both = 0.0f, gloss = 0.0f;
    if (my_token < TOKENS) {
        const int y = g.label[my_token];
        if (y != g.ignore && y >= 0 && y < g.vocab) {
            want = y;
            lse = g.lse[my_token];
            gloss = g.alpha * g.gloss[my_token];
            both = g.alpha * (g.glse ? g.gloss[my_token] + g.glse[my_token] : g.gloss[my_token]);
        }
    }
    // every token's elements of x (zeros for tokens that do not count, whatever they hold) and of gX
    float x[TOKENS][EIGHTS][8], gx[TOKENS][EIGHTS][8];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
        const int y = g.label[t];
        const bool counts = y != g.ignore && y >= 0 && y < g.vocab;
#pragma unroll
        for (int q = 0; q < EIGHTS; ++q) {
            const int h = q * pitch + (int)threadIdx.x * 8;
            Eight<T> e;
            e.load(static_cast<const T *>(g.X) + (counts ? t * g.ldX + h : 0), counts ? g.hidden - h : 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[t][q][i] = e.at(i);
                gx[t][q][i] = 0.0f;
            }
        }
    }

    Eight<T> w[ROWS][EIGHTS], next[ROWS][EIGHTS];
    auto fetch = [&](Eight<T>(&to)[ROWS][EIGHTS], int v0) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int v = v0 + r < g.vocab ? v0 + r : g.vocab - 1;
#pragma unroll
            for (int q = 0; q < EIGHTS; ++q) {
                const int h = q * pitch + (int)threadIdx.x * 8;
                to[r][q].load(W + v * g.ldW + (h < g.hidden ? h : 0), g.hidden - h);
            }
        }
    };
    const int stride = (int)gridDim.x * ROWS;
    int parity = 0;
    fetch(w, blockIdx.x * ROWS);
    for (int v0 = blockIdx.x * ROWS; v0 < g.vocab; v0 += stride) {
        if (v0 + stride < g.vocab) fetch(next, v0 + stride);
        float z[N];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int t = 0; t < PITCH; ++t) {
                float s = 0.0f;
                if (t < TOKENS) {
#pragma unroll
                    for (int q = 0; q < EIGHTS; ++q)
#pragma unroll
                        for (int i = 0; i < 8; ++i) s = fmaf(w[r][q].at(i), x[t][q][i], s);
                }
                z[r * PITCH + t] = s;
            }
        sum_over_wave<N>(z, lane);
        float sum = z[0];
        if (waves > 1) {
            sums[parity][wave][lane] = sum;
            __syncthreads();
            sum = 0.0f;
            for (int k = 0; k < waves; ++k) sum += sums[parity][k][lane];
            parity ^= 1;
        }
        float p = 0.0f;
        if (want >= 0) {
            p = expf(fmaf(g.alpha, sum, -lse)) * both;
            if (v0 + my_row == want) p -= gloss;
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (v0 + r >= g.vocab) break;
            float P[TOKENS];
#pragma unroll
            for (int t = 0; t < TOKENS; ++t)
                P[t] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), (r * PITCH + t) << (6 - LOG)));
#pragma unroll
            for (int q = 0; q < EIGHTS; ++q) {
                const int h = q * pitch + (int)threadIdx.x * 8;
                if (g.part) {
#pragma unroll
                    for (int t = 0; t < TOKENS; ++t)
#pragma unroll
                        for (int i = 0; i < 8; ++i) gx[t][q][i] = fmaf(P[t], w[r][q].at(i), gx[t][q][i]);
                }
                if (g.gW && h < g.hidden) {
                    T *to = static_cast<T *>(g.gW) + (v0 + r) * g.ldGW + h;
                    float out[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) out[i] = P[0] * x[0][q][i];
#pragma unroll
                    for (int t = 1; t < TOKENS; ++t)
#pragma unroll
                        for (int i = 0; i < 8; ++i) out[i] = fmaf(P[t], x[t][q][i], out[i]);
                    if (g.beta != 0.0f) {
                        Eight<T> old;
                        old.load(to, g.hidden - h);
#pragma unroll
                        for (int i = 0; i < 8; ++i) out[i] = fmaf(g.beta, old.at(i), out[i]);
                    }
                    store_eight<T>(to, out, g.hidden - h);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int q = 0; q < EIGHTS; ++q) w[r][q] = next[r][q];
    }
    if (g.part) {
#pragma unroll
        for (int t = 0; t < TOKENS; ++t) {
            float *to = g.part + ((int64_t)blockIdx.x * TOKENS + t) * g.hidden;
#pragma unroll
            for (int q = 0; q < EIGHTS; ++q) {
                const int h = q * pitch + (int)threadIdx.x * 8;
                store_eight<float>(to + h, gx[t][q], g.hidden - h);
            }
        }
    }
}

// gX of the pass above: 64 elements of one token a workgroup, 16 threads with
// four elements each and `slices` (at most 64) of those side by side along the
// parts: one for 16 parts, so that reads in flight hide their latency (1024 parts of
// 5 x 1001: 16 slices 10 us, 64 slices 6.8 us).
template <typename T>
__global__ void __launch_bounds__(1024)
few_gx_kernel(int hidden, int tokens, int vocab, int ignore, const int *__restrict__ label, const float *__restrict__ part,
              int parts, T *gx, int64_t ldgx)
{
    __shared__ float sums[64][64];
    const int slices = blockDim.x >> 4;
    const int t = blockIdx.x, h = blockIdx.y * 64 + (threadIdx.x & 15) * 4, slice = threadIdx.x >> 4, y = label[t];
    const bool counts = y != ignore && y >= 0 && y < vocab;
    const int n = hidden - h;
    vfloat4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    auto one = [&](int k) {
        const float *p = part + ((int64_t)k * tokens + t) * hidden + h;
        vfloat4 a = {0.0f, 0.0f, 0.0f, 0.0f};
        if (n >= 4) {
            a = __builtin_bit_cast(vfloat4, (vint4)*reinterpret_cast<const AnyVector<float>::V *>(p));
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < n) a[e] = p[e];
        }
        return a;
    };
    if (counts) {
        int k = slice;
        for (; k + 7 * slices < parts; k += 8 * slices) {
            vfloat4 a[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) a[u] = one(k + u * slices);
#pragma unroll
            for (int u = 0; u < 8; ++u) v += a[u];
        }
        for (; k < parts; k += slices) v += one(k);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[slice][(threadIdx.x & 15) * 4 + e] = v[e];
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.y * 64 + threadIdx.x < (unsigned)hidden) {
        float s = 0.0f;
#pragma unroll 16
        for (int k = 0; k < slices; ++k) s += sums[k][threadIdx.x];
        gx[t * ldgx + blockIdx.y * 64 + threadIdx.x] = from_float<T>(s);
    }
}

template <typename T, int TOKENS> int launch_few(const FewArgs &g, int parts, hipStream_t stream)
{
    if (g.hidden > 4096) {
        if constexpr (TOKENS <= 4) {
            constexpr int ROWS = sizeof(T) == 2 && TOKENS <= 2 ? 4 : 2;
            hipLaunchKernelGGL((few_kernel<T, TOKENS, 2, ROWS>), dim3(parts), dim3(512), 0, stream, g);
        }
    } else {
        constexpr int ROWS = sizeof(T) == 2 && TOKENS <= 2 ? 8 : 4;
        hipLaunchKernelGGL((few_kernel<T, TOKENS, 1, ROWS>), dim3(parts), dim3((g.hidden + 511) / 512 * 64), 0, stream, g);
    }
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

// Workgroups: two waves for each of the GPU's 1024 SIMDs, as far as there are rows.
int few_parts(int hidden, int vocab)
{
    const int waves = hidden > 4096 ? 8 : (hidden + 511) / 512;
    return (int)std::min<int64_t>(256 * (8 / waves), (vocab + 3) / 4);
}

}  // namespace

// Whether the pass takes a problem: the elements a thread holds have to fit its registers.
bool xent_takes_few(int hidden, int tokens) { return tokens >= 1 && tokens <= 8 && hidden <= (tokens <= 4 ? 8192 : 4096); }

long xent_few_worksize(int hidden, int tokens, int vocab) { return (long)few_parts(hidden, vocab) * tokens * hidden * 4; }

template <typename T>
int xent_few_grad(int hidden, int tokens, int vocab, float alpha, const T *W, int ldW, const T *X, int ldX, const int *label,
                  int ignore, const float *lse, const float *gloss, const float *glse, float beta, T *gW, int ldGW, T *gX,
                  int ldGX, float *work, hipStream_t stream)
{
    const FewArgs f{hidden, vocab, ignore, alpha, beta, W, X, ldW, ldX, ldGW, label, lse, gloss, glse, gW,
                    gX ? work : nullptr};
    const int parts = few_parts(hidden, vocab);
    int rc = ULMBLAS_GPU_BAD_ARGUMENT;
    switch (tokens) {
    case 1: rc = launch_few<T, 1>(f, parts, stream); break;
    case 2: rc = launch_few<T, 2>(f, parts, stream); break;
    case 3: rc = launch_few<T, 3>(f, parts, stream); break;
    case 4: rc = launch_few<T, 4>(f, parts, stream); break;
    case 5: rc = launch_few<T, 5>(f, parts, stream); break;
    case 6: rc = launch_few<T, 6>(f, parts, stream); break;
    case 7: rc = launch_few<T, 7>(f, parts, stream); break;
    case 8: rc = launch_few<T, 8>(f, parts, stream); break;
    }
    if (rc || !gX) return rc;
    const int slices = std::min(std::max(parts / 16, 16), 64);
    hipLaunchKernelGGL(few_gx_kernel<T>, dim3((unsigned)tokens, (unsigned)((hidden + 63) / 64)), dim3(16 * slices), 0, stream, hidden,
                       tokens, vocab, ignore, label, work, parts, gX, (int64_t)ldGX);
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

template int xent_few_grad<float>(int, int, int, float, const float *, int, const float *, int, const int *, int,
                                  const float *, const float *, const float *, float, float *, int, float *, int, float *,
                                  hipStream_t);
template int xent_few_grad<bf16_t>(int, int, int, float, const bf16_t *, int, const bf16_t *, int, const int *, int,
                                   const float *, const float *, const float *, float, bf16_t *, int, bf16_t *, int, float *,
                                   hipStream_t);

}  // namespace ulmgpu
