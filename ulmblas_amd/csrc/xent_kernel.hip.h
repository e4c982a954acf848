// The product kernel behind the softmax cross entropy (xent.hip).
//
// One workgroup computes a BM x BN tile of D = A * B^T with accumulators in
// fp32, for bf16 (v_mfma_f32_32x32x16_bf16) or fp32 (v_mfma_f32_32x32x2_f32)
// operands, and hands it to one of four epilogues:
//
//   STATS  D = logits (A = W: vocabulary rows, B = X: tokens): the running
//          maximum and sum of the softmax over the tile's BM vocabulary rows,
//          per token, and the logit of the label; the logits stay in registers
//   PROB   the same product again, turned into the gradient with respect to
//          the logits, which is stored for the two products below
//   GX     gX^T += W^T * P  (A = W, read along k; B = P)
//   GW     gW^T  = X^T * P  (A = X, B = P, both read along k)
//
// The column of D that a lane of the 32 x 32 MFMA holds is one token (STATS,
// PROB), and its registers run along the vocabulary: the softmax reduces
// inside the lane first, with one exchange between the two halves of the wave
// and one through LDS between the waves of a column.
//
// Operands come in two layouts.  "K-contiguous" rows (W and X in the logits,
// P in GX) are staged as rows of 128 bytes; operands whose k runs across rows
// (W in GX, X and P in GW) are staged as they lie, and the transposition
// happens on the way from LDS to registers (ds_read_b64_tr_b16; fp32 reads
// single words), so no transposed copy of W, X or P exists anywhere.  Both
// kinds travel from global memory straight into LDS, 16 bytes a lane; what
// lies outside the operand is fetched out of the buffer's range, which stores
// zeros.
#ifndef ULMBLAS_XENT_KERNEL_HIP_H
#define ULMBLAS_XENT_KERNEL_HIP_H 1

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

namespace ulmgpu {
namespace xent {

typedef __attribute__((ext_vector_type(2))) int vint2;
typedef __attribute__((ext_vector_type(4))) int vint4;
typedef __attribute__((ext_vector_type(4))) short vshort4;
typedef __attribute__((ext_vector_type(8))) short vshort8;
typedef __attribute__((ext_vector_type(8))) __bf16 vbf8;
typedef __attribute__((ext_vector_type(4))) float vfloat4;
typedef __attribute__((ext_vector_type(16))) float vfloat16;

// bf16 values are carried as their bits.
using bf16_t = unsigned short;

__device__ __forceinline__ float to_float(bf16_t x) { return __uint_as_float((unsigned)x << 16); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
// round to nearest even, NaN stays NaN (v_cvt_pk_bf16_f32)
template <> __device__ __forceinline__ bf16_t from_float<bf16_t>(float x)
{
    return __builtin_bit_cast(unsigned short, (__bf16)x);
}

constexpr int kStepBytes = 128;         // what one step of the k loop takes of a K-contiguous row
template <typename T> constexpr int kStep = kStepBytes / (int)sizeof(T);
constexpr unsigned kOutside = 0x80000000u;      // an offset past every buffer's range

enum Mode { STATS, PROB, GX, GW };

struct ProductArgs {
    const void *A, *B;
    int64_t ldA, ldB;           // bytes from row to row
    int M, N, K;                // rows of D, columns of D, length of the inner products
    int widthA, widthB;         // elements of a row of A / B that exist (K-contiguous: K may end inside a step)
    const int *count;           // tokens with a target: bounds N (STATS, PROB, GX) or K (GW)
    float alpha;
    // STATS
    const int *label;           // per token (compact order)
    float2 *stats;              // [tile of the vocabulary][token]: maximum, sum of exp(z - maximum)
    int64_t ldStats;
    float *target;              // the label's logit
    int first;                  // first vocabulary row of A
    // PROB
    const float *lse, *both, *gloss;    // per token; both = gloss + glse, each times alpha
    void *P;
    int64_t ldP;                // elements
    // GX: partial sums of the splits, each [token][ldD]
    float *part;
    int64_t ldD, splitStride;
    int splits, add;
    // GW
    void *out;
    float beta;
    int wide_out;               // rows of out lie on 16 bytes
};

// Number of 16-byte chunks by which the chunks of row k of an operand that is
// staged along k are rotated (exclusive or), so that the four rows that one
// transposing read takes do not fall on the same banks.
template <int CHUNKS> __device__ __forceinline__ int k_row_swizzle(int k)
{
    if constexpr (CHUNKS >= 16) return (k & 3) * 4;
    return ((k >> 1) & 1) * 4;
}

// The same for K-contiguous rows of 128 bytes: a read takes 16 rows at a time
// from the 64 banks (256 bytes), so pairs of rows get the 8 chunks in turn
// (rotating by the row itself costs every read twice its cycles).
__device__ __forceinline__ int row_swizzle(int row) { return (row >> 1) & 7; }

// Brings R rows (or columns) of one operand for one step into LDS.
template <typename T, int R, bool KC, int WAVES>
struct Loader {
    static constexpr int kBytes = R * kStepBytes;
    static constexpr int kCalls = kBytes / 1024 / WAVES;        // 1024 bytes a wave and call
    static constexpr int kRowBytes = KC ? kStepBytes : R * (int)sizeof(T);
    static constexpr int kChunks = kRowBytes / 16;
    static_assert(kCalls * WAVES * 1024 == kBytes, "the waves share the tile evenly");

    uint64_t base;              // of the tile
    int64_t left;               // bytes of the operand from there on
    int64_t ld;
    unsigned row_offset[kCalls];
    unsigned k_chunk;           // KC: byte inside the step this lane fetches in even calls (odd ones: 64 bytes across)
    unsigned k_bytes;           // KC: bytes of a row that exist

    __device__ void init(const void *p, int64_t ld_, int row0, int rows, int width, int wave, int lane)
    {
        ld = ld_;
        const int64_t total = rows > 0 ? (int64_t)(rows - 1) * ld + (int64_t)width * (int64_t)sizeof(T) : 0;
        const int64_t skip = KC ? (int64_t)row0 * ld : (int64_t)row0 * (int64_t)sizeof(T);
        base = (uint64_t)p + (uint64_t)skip;
        left = total - skip;
        k_bytes = (unsigned)width * (unsigned)sizeof(T);
#pragma unroll
        for (int c = 0; c < kCalls; ++c) {
            const int at = (wave * kCalls + c) * 64 + lane;
            const int row = at / kChunks, chunk = at % kChunks;
            if constexpr (KC) {
                if (c == 0) k_chunk = (unsigned)((chunk ^ row_swizzle(row)) * 16);
                row_offset[c] = (unsigned)(row * ld);
            } else if constexpr (sizeof(T) == 2) {
                row_offset[c] = (unsigned)(row * ld) + (unsigned)((chunk ^ k_row_swizzle<kChunks>(row)) * 16);
            } else {
                row_offset[c] = (unsigned)(row * ld) + (unsigned)(chunk * 16);
            }
        }
    }

    // step s of the k loop into the LDS bytes from `to` on
    __device__ __forceinline__ void fetch(int s, unsigned to, int wave) const
    {
        uint64_t at = base;
        int64_t have = left;
        unsigned k_offset[2] = {0, 0};
        if constexpr (KC) {
            k_offset[0] = (unsigned)s * kStepBytes + k_chunk;
            k_offset[1] = k_offset[0] ^ 64u;
            if (k_offset[0] >= k_bytes) k_offset[0] = kOutside;
            if (k_offset[1] >= k_bytes) k_offset[1] = kOutside;
        } else {
            const int64_t skip = (int64_t)s * kStep<T> * ld;
            at += (uint64_t)skip;
            have -= skip;
        }
        have = have < 0 ? 0 : (have > 0x7fffffff ? 0x7fffffff : have);
        vint4 rsrc;
        rsrc[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
        rsrc[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff);
        rsrc[2] = __builtin_amdgcn_readfirstlane((int)have);
        rsrc[3] = 0x00020000;
#pragma unroll
        for (int c = 0; c < kCalls; ++c) {
            const unsigned lds = __builtin_amdgcn_readfirstlane(to + (unsigned)(wave * kCalls + c) * 1024u);
            const unsigned off = row_offset[c] + k_offset[c & 1];
            // writes LDS only: nothing here has a register for its result
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(lds), "v"(off), "s"(rsrc)
                         : "memory");
        }
    }
};

typedef __attribute__((address_space(3))) const unsigned char lds_byte;

// 16 bytes of operand for one lane: bf16, 8 consecutive k of one row (column);
// fp32, 4 consecutive k.  kk: quarter of the step.
template <typename T, int R, bool KC>
__device__ __forceinline__ vint4 fragment(lds_byte *tile, int r0, int kk, int lane)
{
    if constexpr (KC) {
        const int r = r0 + (lane & 31), g = 2 * kk + (lane >> 5);
        return *(__attribute__((address_space(3))) const vint4 *)(tile + r * kStepBytes + ((g ^ row_swizzle(r)) << 4));
    } else if constexpr (sizeof(T) == 2) {
        constexpr int kChunks = R / 8;
        typedef __attribute__((address_space(3))) vshort4 lds_short4;
        const int m = r0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        vshort8 v;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int k = 16 * kk + 8 * (lane >> 5) + 4 * j + ((lane >> 2) & 3);
            const int at = k * (R * 2) + (((m >> 3) ^ k_row_swizzle<kChunks>(k)) << 4) + (m & 7) * 2;
            const vshort4 h = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(tile + at));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = h[i];
        }
        return __builtin_bit_cast(vint4, v);
    } else {
        vint4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = 8 * kk + 4 * (lane >> 5) + j;
            v[j] = *(__attribute__((address_space(3))) const int *)(tile + (k * R + r0 + (lane & 31)) * 4);
        }
        return v;
    }
}

template <typename T>
__device__ __forceinline__ vfloat16 multiply(vint4 a, vint4 b, vfloat16 c)
{
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vbf8, a), __builtin_bit_cast(vbf8, b), c, 0,
                                                       0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__int_as_float(a[j]), __int_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

// exp(x): bf16 results take the hardware's exponential (its argument is
// rounded at 2^-24 of |x| log2 e, far below bf16), fp32 the library's.
template <typename T> __device__ __forceinline__ float exponential(float x)
{
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
    else return expf(x);
}

// Everything this wave has asked for has arrived, and every wave of the
// workgroup says so.
__device__ __forceinline__ void wait_and_meet()
{
    __builtin_amdgcn_s_waitcnt(0x0070);         // tells the compiler; the next line is what counts
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Spreads the reads of the next quarter's fragments between the matrix
// instructions of this one.
template <int READS, int MFMA, int GROUPS, int I = 0> __device__ __forceinline__ void interleave()
{
    if constexpr (I < GROUPS) {
        __builtin_amdgcn_sched_group_barrier(0x100, (READS * (I + 1)) / GROUPS - (READS * I) / GROUPS, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, (MFMA * (I + 1)) / GROUPS - (MFMA * I) / GROUPS, 0);
        interleave<READS, MFMA, GROUPS, I + 1>();
    }
}

// Which tile of D workgroup `id` computes.  Workgroups go round the 8 XCDs;
// each XCD takes a run of consecutive tiles, ordered in bands of 8 columns, so
// that the 32 tiles its CUs work on at a time are 8 x 4 and share operands in
// its L2.
__device__ __forceinline__ bool tile_of(int id, int tilesM, int tilesN, int &tm, int &tn)
{
    const int tiles = tilesM * tilesN;
    if (id >= tiles) return false;
    const int per = tiles / 8, extra = tiles % 8, x = id % 8;
    id = x * per + (x < extra ? x : extra) + id / 8;
    const int band = id / (8 * tilesM), at = id % (8 * tilesM);
    const int width = tilesN - band * 8 < 8 ? tilesN - band * 8 : 8;
    tn = band * 8 + at % width;
    tm = at / width;
    return true;
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN>
struct Product {
    static constexpr int kWaves = WM * WN;
    static constexpr int kThreads = kWaves * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;      // MFMA tiles of a wave
    static constexpr bool A_KC = MODE == STATS || MODE == PROB, B_KC = MODE != GW;
    // a quarter of a step: LDS reads for its fragments (those staged along k take several), matrix instructions
    static constexpr int kApart = sizeof(T) == 2 ? 2 : 4;
    static constexpr int kReads = TM * (A_KC ? 1 : kApart) + TN * (B_KC ? 1 : kApart);
    static constexpr int kMfma = TM * TN * (sizeof(T) == 2 ? 1 : 4);
    static constexpr int kStage = (BM + BN) * kStepBytes;
    static constexpr int kLds = 2 * kStage;
    using LoadA = Loader<T, BM, A_KC, kWaves>;
    using LoadB = Loader<T, BN, B_KC, kWaves>;

    static __device__ void run(const ProductArgs &g);
};

// The tile of a bf16 result on its way through LDS: rows of BM elements, the
// 16-byte chunks of a row rotated by the row, so that neither the 8-byte writes
// (32 rows at a time) nor the 16-byte reads (along a row) meet on a bank.
template <int BM> __device__ __forceinline__ int staged_at(int row, int col)
{
    constexpr int kChunks = BM / 8;
    return row * (BM * 2) + (((col >> 3) ^ (row & (kChunks - 1))) << 4) + (col & 7) * 2;
}

// Writes the staged tile out, whole rows at a time: rows x cols of it, 16 bytes
// a lane where the rows lie on 16 bytes, else element by element.
template <int BM, int THREADS>
__device__ __forceinline__ void write_staged(const unsigned char *lds, bf16_t *to, int64_t ld, int rows, int cols,
                                             bool wide)
{
    constexpr int kChunks = BM / 8;
    if (wide) {
        for (int i = threadIdx.x; i < rows * kChunks; i += THREADS) {
            const int row = i / kChunks, col = i % kChunks * 8;
            if (col >= cols) continue;
            const vint4 v = *reinterpret_cast<const vint4 *>(lds + staged_at<BM>(row, col));
            bf16_t *p = to + row * ld + col;
            if (col + 8 <= cols) {
                *reinterpret_cast<vint4 *>(p) = v;
            } else {
                for (int e = 0; e < cols - col; ++e) p[e] = reinterpret_cast<const bf16_t *>(&v)[e];
            }
        }
    } else {
        for (int i = threadIdx.x; i < rows * BM; i += THREADS) {
            const int row = i / BM, col = i % BM;
            if (col < cols) to[row * ld + col] = *reinterpret_cast<const bf16_t *>(lds + staged_at<BM>(row, col));
        }
    }
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN>
__device__ void Product<T, MODE, BM, BN, WM, WN>::run(const ProductArgs &g)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds_raw[];
    lds_byte *lds = (lds_byte *)lds_raw;
    const unsigned lds0 = (unsigned)(uintptr_t)lds;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // Columns past the tokens that count have no tile.
    const int live = __builtin_amdgcn_readfirstlane(*g.count);
    const int boundN = MODE == GW ? g.N : (live < g.N ? live : g.N);
    int tm, tn;
    if (!tile_of((int)blockIdx.x, (g.M + BM - 1) / BM, (boundN + BN - 1) / BN, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int K = MODE == GW ? (live < g.K ? live : g.K) : g.K;
    int s0 = 0, s1 = (K + kStep<T> - 1) / kStep<T>;
    if constexpr (MODE == GX) {
        const int steps = s1, z = blockIdx.y;
        s0 = (int)((int64_t)steps * z / g.splits);
        s1 = (int)((int64_t)steps * (z + 1) / g.splits);
    }

    LoadA la;
    LoadB lb;
    // K-contiguous: rows of D's side, of `width` elements; else rows of k
    la.init(g.A, g.ldA, m0, A_KC ? g.M : K, g.widthA, wave, lane);
    lb.init(g.B, g.ldB, n0, B_KC ? g.N : K, g.widthB, wave, lane);

    vfloat16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    // Two halves of LDS, a step each; within a step four quarters, whose fragments are read one quarter ahead.
    // The step changes before the last quarter is multiplied: its fragments are in registers by then, so the
    // half just read can be refilled (for the step after next) and the matrix cores have work while the waves
    // meet and the next step's first fragments come out of LDS.
    if (s0 < s1) {
        la.fetch(s0, lds0, wave);
        lb.fetch(s0, lds0 + BM * kStepBytes, wave);
        vint4 a[2][TM], b[2][TN];
        auto read = [&](int buf, unsigned half, int kk) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                b[buf][j] = fragment<T, BN, B_KC>(lds + half + BM * kStepBytes, (wn * TN + j) * 32, kk, lane);
#pragma unroll
            for (int i = 0; i < TM; ++i)
                a[buf][i] = fragment<T, BM, A_KC>(lds + half, (wm * TM + i) * 32, kk, lane);
        };
        auto quarter = [&](int buf) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = multiply<T>(a[buf][i], b[buf][j], acc[i][j]);
            interleave<kReads, kMfma, (kReads < kMfma ? kReads : kMfma)>();
        };
        wait_and_meet();
        unsigned now = 0;
        if (s0 + 1 < s1) {
            la.fetch(s0 + 1, lds0 + kStage, wave);
            lb.fetch(s0 + 1, lds0 + kStage + BM * kStepBytes, wave);
        }
        read(0, now, 0);
        auto first_three = [&] {
#pragma unroll
            for (int kk = 0; kk < 3; ++kk) {
                read((kk + 1) & 1, now, kk + 1);
                quarter(kk & 1);
            }
        };
        for (int s = s0; s + 1 < s1; ++s) {
            first_three();
            wait_and_meet();
            if (s + 2 < s1) {
                la.fetch(s + 2, lds0 + now, wave);
                lb.fetch(s + 2, lds0 + now + BM * kStepBytes, wave);
            }
            now = kStage - now;
            read(0, now, 0);
            quarter(1);
        }
        first_three();
        quarter(1);
    }

    const int mw = m0 + wm * TM * 32 + (lane >> 5) * 4, nw = n0 + wn * TN * 32 + (lane & 31);
    if constexpr (MODE == STATS) {
        wait_and_meet();
        float2 *red = reinterpret_cast<float2 *>(lds_raw);      // [wm][column]
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 32;
            const int want = n < boundN ? g.label[n] - g.first : -1;
            float top = -INFINITY, hit = 0.0f;
            bool has = false;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = mw + i * 32 + (r >> 2) * 8 + (r & 3);
                    const float z = m < g.M ? g.alpha * acc[i][j][r] : -INFINITY;
                    acc[i][j][r] = z;
                    top = fmaxf(top, z);
                    if (m == want && m < g.M) {
                        hit = z;
                        has = true;
                    }
                }
            if (has) g.target[n] = hit;
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += exponential<T>(acc[i][j][r] - from);
            sum += __shfl_xor(sum, 32);
            if (lane < 32) red[wm * BN + (wn * TN + j) * 32 + lane] = make_float2(top, sum);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BN; c += kThreads) {
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WM; ++w) top = fmaxf(top, red[w * BN + c].x);
            const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < WM; ++w) {
                const float t = red[w * BN + c].x;
                sum += red[w * BN + c].y * exponential<T>((t == -INFINITY ? 0.0f : t) - from);
            }
            if (n0 + c < boundN) g.stats[(int64_t)tm * g.ldStats + n0 + c] = make_float2(top, sum);
        }
    } else if constexpr (MODE == PROB) {
        // Rounded to the operands' type, since the two products that follow run on it: each element is off by
        // at most half a step (bf16: 2^-9 of itself), and the sums over tokens or vocabulary average that out.
        T *P = static_cast<T *>(g.P);
        if constexpr (sizeof(T) == 2) wait_and_meet();
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 32;
            if (n >= boundN) continue;
            const float lse = g.lse[n], both = g.both[n], gloss = g.gloss[n];
            const int want = g.label[n] - g.first;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = mw + i * 32 + q * 8;
                    T v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float p = exponential<T>(g.alpha * acc[i][j][4 * q + r] - lse) * both;
                        if (m + r == want) p -= gloss;
                        v[r] = from_float<T>(m + r < g.M ? p : 0.0f);
                    }
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<vint2 *>(lds_raw + staged_at<BM>(n - n0, m - m0)) =
                            *reinterpret_cast<vint2 *>(v);
                    } else {
                        *reinterpret_cast<vint4 *>(P + (int64_t)n * g.ldP + m) = *reinterpret_cast<vint4 *>(v);
                    }
                }
        }
        if constexpr (sizeof(T) == 2) {
            __syncthreads();
            write_staged<BM, kThreads>(lds_raw, P + (int64_t)n0 * g.ldP + m0, g.ldP,
                                       boundN - n0 < BN ? boundN - n0 : BN, BM, true);
        }
    } else if constexpr (MODE == GX) {
        float *part = g.part + (int64_t)blockIdx.y * g.splitStride;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 32;
            if (n >= boundN) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = mw + i * 32 + q * 8;
                    if (m >= g.M) continue;         // ldD is a multiple of 4: four fit where one does
                    vfloat4 *to = reinterpret_cast<vfloat4 *>(part + (int64_t)n * g.ldD + m);
                    vfloat4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if (g.add) {
                        const vfloat4 old = *to;
                        v += old;
                    }
                    *to = v;
                }
        }
    } else {
        T *out = static_cast<T *>(g.out);
        if constexpr (sizeof(T) == 2) wait_and_meet();
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 32;
            if (n >= boundN) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int m = mw + i * 32 + q * 8;
                    T *to = out + (int64_t)n * g.ldD + m;
                    float x[4];
                    T v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = acc[i][j][4 * q + r];
                        if (g.beta != 0.0f && m + r < g.M) x[r] += g.beta * to_float(to[r]);
                        v[r] = from_float<T>(x[r]);
                    }
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<vint2 *>(lds_raw + staged_at<BM>(n - n0, m - m0)) =
                            *reinterpret_cast<vint2 *>(v);
                    } else if (g.wide_out && m + 4 <= g.M) {
                        *reinterpret_cast<vint4 *>(to) = *reinterpret_cast<vint4 *>(v);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (m + r < g.M) to[r] = v[r];
                    }
                }
        }
        if constexpr (sizeof(T) == 2) {
            __syncthreads();
            write_staged<BM, kThreads>(lds_raw, out + (int64_t)n0 * g.ldD + m0, g.ldD, g.N - n0 < BN ? g.N - n0 : BN,
                                       g.M - m0 < BM ? g.M - m0 : BM, g.wide_out);
        }
    }
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM *WN * 64, 2)
product_kernel(ProductArgs g)
{
    Product<T, MODE, BM, BN, WM, WN>::run(g);
}

}  // namespace xent
}  // namespace ulmgpu
#endif
