// The Euclidean norm of a group of tensors taken as one vector, and the group
// scaled down to a largest norm: nrm2 and scal over the gradients of a model.
//
// The list of tensors travels in the kernel arguments, kGroup of them a launch:
// nothing is copied to the device, so a call may be recorded into a graph and
// the caller's arrays are free as soon as it returns.  A group is cut into
// chunks of equal length; a workgroup takes every gridDim-th chunk, finds the
// tensor it lies in and sums its squares in fp64, which neither overflows nor
// underflows for any fp32 or bf16 value and leaves nothing of the rounding of a
// long sum.  One more workgroup adds the partial sums in a fixed order: the
// same call gives the same bits.
#include "internal.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <vector>

using namespace ulmgpu;

namespace ulmgpu {
namespace {

typedef __attribute__((ext_vector_type(4))) unsigned vuint4;

constexpr int kGroup = 128;             // tensors a launch
constexpr int kBlocks = 2048;           // workgroups a launch at the most (8 a CU), a partial sum each
constexpr int kThreads = 256;

struct GroupArgs {
    const void *x[kGroup];
    void *y[kGroup];
    int64_t n[kGroup];
    unsigned first[kGroup + 1];         // chunks before each tensor; [count]: all
    unsigned type[kGroup / 32];         // bit set: bf16
    int count;
    int chunk;                          // elements
};

__device__ __forceinline__ int tensor_of(const GroupArgs &g, unsigned chunk)
{
    int lo = 0, hi = g.count - 1;       // the last tensor whose first chunk is not beyond
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (g.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T> struct Wide;      // 16 bytes at whatever address the elements have
template <> struct Wide<float> { typedef vuint4 V __attribute__((aligned(4))); };
template <> struct Wide<unsigned short> { typedef vuint4 V __attribute__((aligned(2))); };

__device__ __forceinline__ void add_squares(vuint4 v, float, double &s0, double &s1)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double d = __uint_as_float(v[i]);
        (i & 1 ? s1 : s0) += d * d;
    }
}
__device__ __forceinline__ void add_squares(vuint4 v, unsigned short, double &s0, double &s1)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double a = __uint_as_float(v[i] << 16), b = __uint_as_float(v[i] & 0xffff0000u);
        s0 += a * a;
        s1 += b * b;
    }
}
__device__ __forceinline__ double value(const float *p) { return *p; }
__device__ __forceinline__ double value(const unsigned short *p) { return __uint_as_float((unsigned)*p << 16); }

// squares of x[0 .. n)
template <typename T> __device__ __forceinline__ double chunk_squares(const T *x, int n)
{
    constexpr int V = 16 / sizeof(T);
    double s0 = 0.0, s1 = 0.0;
    const int head = std::min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    if ((int)threadIdx.x < head) s0 = value(x + threadIdx.x) * value(x + threadIdx.x);
    const int vectors = (n - head) / V;
    const vuint4 *p = reinterpret_cast<const vuint4 *>(x + head);
    int i = threadIdx.x;
    for (; i + 3 * kThreads < vectors; i += 4 * kThreads) {
        vuint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = p[i + u * kThreads];
#pragma unroll
        for (int u = 0; u < 4; ++u) add_squares(v[u], T(), s0, s1);
    }
    for (; i < vectors; i += kThreads) add_squares(p[i], T(), s0, s1);
    const int rest = head + vectors * V + threadIdx.x;
    if (rest < n) s1 += value(x + rest) * value(x + rest);
    return s0 + s1;
}

__device__ double block_sum(double s)
{
    __shared__ double part[16];
    for (int d = 32; d; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (unsigned w = 0; w < blockDim.x / 64; ++w) s += part[w];
    return s;
}

__global__ void __launch_bounds__(kThreads) squares_kernel(GroupArgs g, double *partial)
{
    double s = 0.0;
    for (unsigned c = blockIdx.x; c < g.first[g.count]; c += gridDim.x) {
        const int i = tensor_of(g, c);
        const int64_t at = (int64_t)(c - g.first[i]) * g.chunk;
        const int n = (int)std::min<int64_t>(g.chunk, g.n[i] - at);
        s += g.type[i / 32] >> (i % 32) & 1 ? chunk_squares(static_cast<const unsigned short *>(g.x[i]) + at, n)
                                            : chunk_squares(static_cast<const float *>(g.x[i]) + at, n);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ void __launch_bounds__(1024) norm_kernel(const double *partial, int count, float *norm)
{
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 1024) s += partial[i];
    s = block_sum(s);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

__device__ __forceinline__ vuint4 scaled(vuint4 v, float f, float)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    return v;
}
__device__ __forceinline__ unsigned bf16_bits(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ __forceinline__ vuint4 scaled(vuint4 v, float f, unsigned short)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = bf16_bits(__uint_as_float(v[i] << 16) * f) | bf16_bits(__uint_as_float(v[i] & 0xffff0000u) * f) << 16;
    return v;
}
__device__ __forceinline__ void scale_one(const float *x, float *y, float f) { *y = *x * f; }
__device__ __forceinline__ void scale_one(const unsigned short *x, unsigned short *y, float f)
{
    *y = (unsigned short)bf16_bits(__uint_as_float((unsigned)*x << 16) * f);
}

// Vectors lie on 16 bytes of y; x may start anywhere.
template <typename T> __device__ __forceinline__ void chunk_scale(const T *x, T *y, int n, float f)
{
    constexpr int V = 16 / sizeof(T);
    using XV = typename Wide<T>::V;
    const int head = std::min(n, (int)((16 - ((uintptr_t)y & 15)) & 15) / (int)sizeof(T));
    if ((int)threadIdx.x < head) scale_one(x + threadIdx.x, y + threadIdx.x, f);
    const int vectors = (n - head) / V;
    const XV *p = reinterpret_cast<const XV *>(x + head);
    vuint4 *q = reinterpret_cast<vuint4 *>(y + head);
    int i = threadIdx.x;
    for (; i + 3 * kThreads < vectors; i += 4 * kThreads) {
        vuint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = p[i + u * kThreads];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[i + u * kThreads] = scaled(v[u], f, T());
    }
    for (; i < vectors; i += kThreads) q[i] = scaled((vuint4)p[i], f, T());
    const int rest = head + vectors * V + threadIdx.x;
    if (rest < n) scale_one(x + rest, y + rest, f);
}

__global__ void __launch_bounds__(kThreads) clip_kernel(GroupArgs g, const float *norm, float largest)
{
    // a norm that is no number or infinite leaves the group as it is: the caller sees it in the norm
    const float have = *norm;
    const float f = have > largest && have < INFINITY ? largest / have : 1.0f;
    for (unsigned c = blockIdx.x; c < g.first[g.count]; c += gridDim.x) {
        const int i = tensor_of(g, c);
        if (f == 1.0f && g.x[i] == g.y[i]) continue;
        const int64_t at = (int64_t)(c - g.first[i]) * g.chunk;
        const int n = (int)std::min<int64_t>(g.chunk, g.n[i] - at);
        if (g.type[i / 32] >> (i % 32) & 1) {
            chunk_scale(static_cast<const unsigned short *>(g.x[i]) + at, static_cast<unsigned short *>(g.y[i]) + at, n,
                        f);
        } else {
            chunk_scale(static_cast<const float *>(g.x[i]) + at, static_cast<float *>(g.y[i]) + at, n, f);
        }
    }
}

constexpr int64_t kMaxLength = (int64_t)1 << 40;

int bad(const char *text)
{
    g_last_error = text;
    return ULMBLAS_GPU_BAD_ARGUMENT;
}

int check(int count, const char *type, const long *n, const void *const *x)
{
    if (count < 0) return bad("negative count");
    if (count > 0 && (!type || !n || !x)) return bad("null list");
    for (int i = 0; i < count; ++i) {
        if (type[i] != 's' && type[i] != 'b') return bad("unknown type");
        if (n[i] < 0 || n[i] > kMaxLength) return bad("invalid length");
        if (n[i] > 0 && !x[i]) return bad("null tensor");
        if ((uintptr_t)x[i] % (type[i] == 's' ? 4 : 2)) return bad("tensor off its type's alignment");
    }
    return ULMBLAS_GPU_OK;
}

// Whether the tensors written overlap neither each other nor the norm nor any that is read, but for the one with the same
// number, which may be the same memory.  (60 tensors: 1 us of the host's time.)
int check_apart(int count, const char *type, const long *n, const void *const *x, void *const *y, const float *norm)
{
    struct Span {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Span> spans;
    try {
        spans.reserve(2 * (size_t)count + 1);
    } catch (const std::exception &) {
        return bad("out of host memory");
    }
    spans.push_back({(uintptr_t)norm, (uintptr_t)(norm + 1), false});
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)n[i] * (type[i] == 's' ? 4 : 2), from = (uintptr_t)x[i], to = (uintptr_t)y[i];
        spans.push_back({to, to + bytes, true});
        if (from != to) spans.push_back({from, from + bytes, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    uintptr_t all = 0, written = 0;         // ends of the spans so far
    for (const Span &s : spans) {
        if (s.from < (s.written ? all : written)) return bad("a tensor that is written overlaps another one or the norm");
        all = std::max(all, s.to);
        if (s.written) written = std::max(written, s.to);
    }
    return ULMBLAS_GPU_OK;
}

int launches(int count) { return (count + kGroup - 1) / kGroup; }

// The tensors from `from` on, as many as a launch takes; returns how many
// workgroups that is.  Chunks are as long as gives every workgroup of a full
// grid one, between 2048 and 32768 elements.
unsigned fill(GroupArgs &g, int from, int count, const char *type, const long *n, const void *const *x, void *const *y)
{
    g = GroupArgs{};
    g.count = std::min(kGroup, count - from);
    int64_t all = 0;
    for (int i = 0; i < g.count; ++i) all += n[from + i];
    int64_t chunk = std::min<int64_t>(32768, std::max<int64_t>(2048, (all / kBlocks + 2047) / 2048 * 2048));
    while ((all / chunk) + g.count > 0x7fffffff) chunk *= 2;
    g.chunk = (int)chunk;
    unsigned chunks = 0;
    for (int i = 0; i < g.count; ++i) {
        g.x[i] = x[from + i];
        g.y[i] = y ? y[from + i] : nullptr;
        g.n[i] = n[from + i];
        g.first[i] = chunks;
        if (type[from + i] == 'b') g.type[i / 32] |= 1u << (i % 32);
        chunks += (unsigned)((n[from + i] + chunk - 1) / chunk);
    }
    g.first[g.count] = chunks;
    return std::min<unsigned>(kBlocks, chunks);
}

}  // namespace
}  // namespace ulmgpu

extern "C" {

long ulmblas_gpu_gnrm2_worksize(int count)
{
    return (long)std::max(1, launches(std::max(count, 0))) * kBlocks * (long)sizeof(double);
}

int ulmblas_gpu_gnrm2(int count, const char *type, const long *n, const void *const *dX, float *dNorm, void *work,
                      void *stream_)
{
    const int rc = check(count, type, n, dX);
    if (rc) return rc;
    if (!dNorm || !work) return bad("null result or workspace");
    if ((uintptr_t)work & 7) return bad("workspace not on 8 bytes");
    const uintptr_t from = (uintptr_t)work, to = from + (uintptr_t)ulmblas_gpu_gnrm2_worksize(count);
    for (int i = 0; i < count; ++i) {
        const uintptr_t x = (uintptr_t)dX[i];
        if (n[i] > 0 && x < to && from < x + (uintptr_t)n[i] * (type[i] == 's' ? 4 : 2))
            return bad("the workspace overlaps a tensor");
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    double *partial = static_cast<double *>(work);
    int sums = 0;
    GroupArgs g;
    for (int from = 0; from < count; from += kGroup) {
        const unsigned blocks = fill(g, from, count, type, n, dX, nullptr);
        if (blocks == 0) continue;
        hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kThreads), 0, stream, g, partial + sums);
        HIP_TRY(hipGetLastError());
        sums += (int)blocks;
    }
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(1024), 0, stream, partial, sums, dNorm);
    HIP_TRY(hipGetLastError());
    return ULMBLAS_GPU_OK;
}

int ulmblas_gpu_gclip(int count, const char *type, const long *n, const void *const *dX, void *const *dY,
                      const float *dNorm, float largest, void *stream_)
{
    int rc = check(count, type, n, dX);
    if (rc) return rc;
    if ((rc = check(count, type, n, dY))) return rc;
    if (!(largest >= 0.0f)) return bad("largest norm negative or no number");
    if (count == 0) return ULMBLAS_GPU_OK;
    if (!dNorm) return bad("null norm");
    if ((rc = check_apart(count, type, n, dX, dY, dNorm))) return rc;
    GroupArgs g;
    for (int from = 0; from < count; from += kGroup) {
        const unsigned blocks = fill(g, from, count, type, n, dX, dY);
        if (blocks == 0) continue;
        hipLaunchKernelGGL(clip_kernel, dim3(blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream_), g, dNorm,
                           largest);
        HIP_TRY(hipGetLastError());
    }
    return ULMBLAS_GPU_OK;
}

}  // extern "C"
