// The product kernel behind the softmax cross entropy (xent.hip).
//
// One workgroup computes a BM x BN tile of D = A * B^T with accumulators in
// fp32, for bf16 (v_mfma_f32_16x16x32_bf16) or fp32 (v_mfma_f32_16x16x4_f32)
// operands, and hands it to one of four epilogues:
//
//   STATS  D = logits (A = W: vocabulary rows, B = X: tokens): the running
//          maximum and sum of the softmax over the tile's BM vocabulary rows,
//          per token, and the logit of the label; the logits stay in registers
//   PROB   the same product again, turned into the gradient with respect to
//          the logits, P, which is stored for the two products below
//   GX     gX^T += W^T * P  (A = W, read along k; B = P)
//   GW     gW^T  = X^T * P  (A = X, B = P, both read along k)
//
// The column of D that a lane of the MFMA holds is one token (STATS, PROB), and
// its registers run along the vocabulary: the softmax reduces inside the lane
// first, with two exchanges between the lanes of a column and one through LDS
// between the waves of a column.
//
// Operands come in two layouts.  "K-contiguous" rows (W and X in the logits,
// P in GX) are staged as rows of 128 bytes; operands whose k runs across rows
// (W in GX, X and P in GW) are staged as they lie, and the transposition
// happens on the way from LDS to registers (ds_read_b64_tr_b16; fp32 reads
// single words), so no transposed copy of W, X or P exists anywhere.  Both
// kinds travel from global memory straight into LDS, 16 bytes a lane; what
// lies outside the operand is fetched out of the buffer's range, which stores
// zeros.
//
// P is kept in blocks of 256 tokens by 128 bytes of vocabulary, 32 KB without
// a gap, so that what GX takes of it in one step is one such block and what GW
// takes is 8 KB at a time (rows of P 128 KB apart: 3.53 ms for the GX product
// 4096 x 8192 x 65536, in blocks 3.32 ms).
//
// Measured on bf16 tiles of 256 x 256 (tokens x hidden x vocabulary): the matrix
// cores are busy 58 - 66 % of the cycles on 8192 x 4096 x 131072 and 35 - 57 % on
// 2048 x 2048 x 32768, half masked (GW the least: 16 steps a tile), at the 1.5 -
// 2.1 GHz that the power limit leaves.  16 x 16 MFMAs run at a higher clock than
// 32 x 32 ones (they read and write half the accumulators per product): STATS
// 1.90 -> 1.81 ms (8192 x 4096 x 32768).
#ifndef ULMBLAS_XENT_KERNEL_HIP_H
#define ULMBLAS_XENT_KERNEL_HIP_H 1

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace ulmgpu {
namespace xent {

typedef __attribute__((ext_vector_type(2))) int vint2;
typedef __attribute__((ext_vector_type(4))) int vint4;
typedef __attribute__((ext_vector_type(4))) short vshort4;
typedef __attribute__((ext_vector_type(8))) short vshort8;
typedef __attribute__((ext_vector_type(8))) __bf16 vbf8;
typedef __attribute__((ext_vector_type(4))) float vfloat4;

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

// blocks of P
constexpr int kBlockTokens = 256, kBlockBytes = kBlockTokens * kStepBytes;

enum Mode { STATS, PROB, GX, GW };

// How an operand lies in memory: rows along k; rows across k; P, taken along
// the vocabulary (its k) or across the tokens (its k).
enum Lie { ALONG, ACROSS, P_ALONG, P_ACROSS };
constexpr bool k_contiguous(Lie lie) { return lie == ALONG || lie == P_ALONG; }

struct ProductArgs {
    const void *A, *B;
    int64_t ldA, ldB;           // bytes from row to row (P: from one row of blocks to the next)
    int M, N, K;                // rows of D, columns of D, length of the inner products
    int widthA, widthB;         // elements of a row of A / B that exist (P: blocks in all)
    const int *count;           // tokens with a target: bounds N (STATS, PROB, GX) or K (GW)
    float alpha;
    const int *label;           // per token (compact order)
    int first;                  // first vocabulary row of A (STATS, PROB) or column of D (GW)
    // STATS
    float2 *stats;              // [tile of the vocabulary][token]: maximum, sum of exp(z - maximum)
    int64_t ldStats;
    float *target;              // the label's logit
    // PROB
    const float *lse, *both, *gloss;    // per token; both = gloss + glse, each times alpha
    void *P;
    int64_t ldP;                // bytes from one row of blocks to the next
    const int *rank;            // per token: its place in `member` (null: the tokens are too few to be sorted)
    float *delta;               // per place there: what rounding took from P at the label (PROB writes, GW reads)
    // GX: partial sums of the splits, each [token][ldD], one after the other as long as `count` makes them
    float *part;
    int64_t ldD;                // elements; GW: of out
    int groups, steps, add;     // workgroups to spread over, steps of k of a whole piece; whether there are sums to add to
    // GW
    void *out;
    float beta;
    bool past;                  // bf16's gW goes past the caches (kPastCaches)
    const int *bucket;          // first place of each group of 128 vocabulary rows
    const int2 *member;         // tokens (compact) in the order of their label's group, and their labels
};

// Chunks of 16 bytes of an operand staged across k are rotated (exclusive or) by
// its row, so that the rows that one read takes (four groups of lanes, four rows
// each in bf16) spread over the 64 banks.
template <typename T, int CHUNKS> __device__ __forceinline__ int across_swizzle(int k)
{
    if constexpr (sizeof(T) == 2) return ((k & 3) * 4 + ((k >> 3) & 1) * 2) & (CHUNKS - 1);
    return ((k >> 2) & 3) * 4;
}

// The same for K-contiguous rows of 128 bytes: a read takes 16 rows at a time
// from the 64 banks (256 bytes), so pairs of rows get the 8 chunks in turn
// (rotating by the row itself costs every read twice its cycles).
__device__ __forceinline__ int row_swizzle(int row) { return (row >> 1) & 7; }

// 16 bytes at whatever address its elements have.
template <typename T> struct AnyVector;
template <> struct AnyVector<bf16_t> { typedef vint4 V __attribute__((aligned(2))); };
template <> struct AnyVector<float> { typedef vint4 V __attribute__((aligned(4))); };

// Brings R rows (or columns) of one operand for one step into LDS.
template <typename T, int R, Lie LIE, int WAVES>
struct Loader {
    static constexpr int kBytes = R * kStepBytes;
    static constexpr int kCalls = kBytes / 1024 / WAVES;        // 1024 bytes a wave and call
    static constexpr bool kAlong = k_contiguous(LIE);
    static constexpr int kRowBytes = kAlong ? kStepBytes : R * (int)sizeof(T);
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kStepsPerBlock = kBlockTokens / kStep<T>;
    static_assert(kCalls * WAVES * 1024 == kBytes, "the waves share the tile evenly");

    vint4 held[kCalls];         // take() / put()
    uint64_t base;              // of the tile
    int64_t left;               // bytes of the operand from there on
    int64_t ld;
    unsigned row_offset[kCalls];
    unsigned k_chunk;           // ALONG: byte inside the step this lane fetches in even calls (odd ones: 64 across)
    unsigned k_bytes;           // ALONG: bytes of a row that exist

    // WORD: what the last row may be rounded up to (4 bytes for calls, nothing for take())
    template <int64_t WORD = 4>
    __device__ void init(const void *p, int64_t ld_, int row0, int rows, int width, int wave, int lane)
    {
        ld = ld_;
        int64_t total, skip;
        if constexpr (LIE == ALONG || LIE == ACROSS) {
            // whole words: the buffer's range would cut off half of an odd row's last one
            total = rows > 0 ? ((int64_t)(rows - 1) * ld + (int64_t)width * (int64_t)sizeof(T) + WORD - 1) & -WORD : 0;
            skip = LIE == ALONG ? (int64_t)row0 * ld : (int64_t)row0 * (int64_t)sizeof(T);
        } else {
            total = (int64_t)width * kBlockBytes;
            skip = LIE == P_ALONG ? (row0 / kBlockTokens) * ld + (row0 % kBlockTokens) * kStepBytes
                                  : (int64_t)(row0 / kStep<T>) * kBlockBytes;
        }
        base = (uint64_t)p + (uint64_t)skip;
        left = total - skip;
        k_bytes = (unsigned)width * (unsigned)sizeof(T);
#pragma unroll
        for (int c = 0; c < kCalls; ++c) {
            const int at = (wave * kCalls + c) * 64 + lane;
            const int row = at / kChunks, chunk = at % kChunks;
            if constexpr (LIE == ALONG) {
                if (c == 0) k_chunk = (unsigned)((chunk ^ row_swizzle(row)) * 16);
                row_offset[c] = (unsigned)(row * ld);
            } else if constexpr (LIE == P_ALONG) {
                row_offset[c] = (unsigned)(row * kStepBytes + (chunk ^ row_swizzle(row)) * 16);
            } else {
                const int from = chunk ^ across_swizzle<T, kChunks>(row);
                row_offset[c] = LIE == ACROSS ? (unsigned)(row * ld) + (unsigned)(from * 16)
                                              : (unsigned)(from / 8 * kBlockBytes + row * kStepBytes + from % 8 * 16);
            }
        }
    }

    // step s of the k loop: the buffer and the offsets its calls use
    __device__ __forceinline__ void aim(int s, int end, vint4 &rsrc, unsigned (&k_offset)[2]) const
    {
        int64_t skip = 0;
        k_offset[0] = k_offset[1] = 0;
        if constexpr (LIE == ALONG) {
            k_offset[0] = (unsigned)s * kStepBytes + k_chunk;
            k_offset[1] = k_offset[0] ^ 64u;
            if (k_offset[0] >= k_bytes) k_offset[0] = kOutside;
            if (k_offset[1] >= k_bytes) k_offset[1] = kOutside;
        } else if constexpr (LIE == ACROSS) {
            skip = (int64_t)s * kStep<T> * ld;
        } else if constexpr (LIE == P_ALONG) {
            skip = (int64_t)s * kBlockBytes;
        } else {
            skip = (int64_t)(s / kStepsPerBlock) * ld + s % kStepsPerBlock * (kStep<T> * kStepBytes);
        }
        const uint64_t at = base + (uint64_t)skip;
        int64_t have = left - skip;
        have = have < 0 || s >= end ? 0 : (have > 0x7fffffff ? 0x7fffffff : have);
        rsrc[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
        rsrc[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xffff);
        rsrc[2] = __builtin_amdgcn_readfirstlane((int)have);
        rsrc[3] = 0x00020000;
    }

    // call c of a step into the tile at LDS byte `to`; writes LDS only: nothing here has a register for its result
    __device__ __forceinline__ void call(int c, vint4 rsrc, const unsigned (&k_offset)[2], unsigned to, int wave) const
    {
        const unsigned lds = __builtin_amdgcn_readfirstlane(to + (unsigned)(wave * kCalls + c) * 1024u);
        const unsigned off = row_offset[c] + k_offset[c & 1];
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(lds), "v"(off), "s"(rsrc)
                     : "memory");
    }

    // The same through registers, for operands whose rows start on any element: all calls of step s, and their tile.
    __device__ __forceinline__ void take(int s)
    {
        vint4 rsrc;
        unsigned k_offset[2];
        aim(s, s + 1, rsrc, k_offset);
        const int64_t skip = (int64_t)(((uint64_t)(uint32_t)rsrc[1] << 32 | (uint32_t)rsrc[0]) - (base & 0xffffffffffffull));
        const unsigned have = (unsigned)rsrc[2];
#pragma unroll
        for (int c = 0; c < kCalls; ++c) {
            const unsigned off = row_offset[c] + k_offset[c & 1];
            const T *p = reinterpret_cast<const T *>(base + (uint64_t)skip + off);
            held[c] = vint4{0, 0, 0, 0};
            if (off < have && have - off >= 16) {
                held[c] = *reinterpret_cast<const typename AnyVector<T>::V *>(p);
            } else if (off < have) {            // the operand ends inside the chunk
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(T); ++e) {
                    if (e * sizeof(T) >= have - off) continue;
                    if constexpr (sizeof(T) == 2) held[c][e >> 1] |= (int)((unsigned)p[e] << 16 * (e & 1));
                    else held[c][e] = __float_as_int(p[e]);
                }
            }
        }
    }
    __device__ __forceinline__ void put(unsigned char *to, int wave, int lane) const
    {
#pragma unroll
        for (int c = 0; c < kCalls; ++c) *reinterpret_cast<vint4 *>(to + (wave * kCalls + c) * 1024 + lane * 16) = held[c];
    }
};

typedef __attribute__((address_space(3))) const unsigned char lds_byte;

// Fragments: 16 bytes of operand for one lane (bf16: 8 consecutive k of one row
// or column; fp32: 4).  base() is the byte in the tile from which this lane
// reads the first fragment of its wave, read() fragment x (16 rows on) of half
// kk of the step.  The rotations of the chunks touch bits of the address that x
// and kk own alone, so a fragment is an exclusive or and a constant away.
template <typename T, int R, bool KC> struct Fragment {
    static __device__ __forceinline__ unsigned base(int first, int lane)
    {
        if constexpr (KC) {
            const int r = first + (lane & 15);
            return (unsigned)(r * kStepBytes + (((lane >> 4) ^ row_swizzle(r)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            const int m = first + (lane & 3) * 4, k = 8 * (lane >> 4) + ((lane >> 2) & 3);
            return (unsigned)(k * (R * 2) + (((m >> 3) ^ across_swizzle<T, R / 8>(k)) << 4) + (m & 7) * 2);
        } else {
            const int m = first + (lane & 15), k = 4 * (lane >> 4);
            return (unsigned)(k * (R * 4) + (((m >> 2) ^ across_swizzle<T, R / 4>(k)) << 4) + (m & 3) * 4);
        }
    }
    static __device__ __forceinline__ vint4 read(lds_byte *tile, unsigned base, int x, int kk)
    {
        if constexpr (KC) {
            return *(__attribute__((address_space(3))) const vint4 *)(tile + (base ^ (unsigned)(kk << 6)) + x * (16 * kStepBytes));
        } else if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) vshort4 lds_short4;
            vshort8 v;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const vshort4 h = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_short4 *)(tile + (base ^ (unsigned)(x << 5)) + (32 * kk + 4 * j) * (R * 2)));
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * j + i] = h[i];
            }
            return __builtin_bit_cast(vint4, v);
        } else {
            vint4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = *(__attribute__((address_space(3))) const int *)(tile + (base ^ (unsigned)(x << 6)) +
                                                                       (16 * kk + j) * (R * 4));
            return v;
        }
    }
};

// Which of a fragment's 16 bytes hold k that exist, `have` elements from its first on.
template <typename T> __device__ __forceinline__ vint4 valid_k(int have)
{
    vint4 v;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 2) v[w] = have > 2 * w + 1 ? -1 : have > 2 * w ? 0xffff : 0;
        else v[w] = have > w ? -1 : 0;
    }
    return v;
}

// One row of tiles: c[j] += a * b[j].  fp32 takes the four k of a fragment one
// after the other for all tiles, so that no matrix instruction waits for the
// one before it.
template <typename T, int TN>
__device__ __forceinline__ void multiply(vint4 a, const vint4 (&b)[TN], vfloat4 (&c)[TN])
{
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
            c[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vbf8, a), __builtin_bit_cast(vbf8, b[j]),
                                                           c[j], 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                c[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[e]), __int_as_float(b[j][e]), c[j], 0, 0, 0);
    }
}

// exp(scale * x): for bf16 the hardware's exponential with log2 e in the scale
// (its argument is rounded at 2^-24 of itself, far below bf16), for fp32 the
// library's.
template <typename T> __device__ __forceinline__ float scale_of(float alpha)
{
    return sizeof(T) == 2 ? alpha * 1.4426950408889634f : alpha;
}
template <typename T> __device__ __forceinline__ float exponential(float x)
{
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(x);
    else return expf(x);
}

// All but the OPEN latest fetches of this wave have arrived, it has read all it
// asked LDS for, and every wave of the workgroup says so.
template <int OPEN = 0> __device__ __forceinline__ void wait_and_meet()
{
    static_assert(OPEN < 64, "six bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | (OPEN & 15) | (OPEN >> 4) << 14);       // tells the compiler; the next line is what counts
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(OPEN) : "memory");
}

// Into how many parts GX cuts its k, up to `groups` workgroups: where the CU with
// the most parts is done first.  In steps of k: a part has its share of them and
// about 6 for beginning and end, and every part costs its sums written and read
// again, 8 bytes for each element of gX (a step of the 256 x 256 tile takes as
// long as 650000 of them).  All 64 lanes of a wave take part, one possibility
// each; the answer depends on the arguments alone.
constexpr int kMaxSplits = 64;
__device__ __forceinline__ int splits_of(int groups, int tiles, int steps, int live, int hidden)
{
    const int lane = threadIdx.x & 63, n = lane + 1;
    float cost = INFINITY;
    if (n == 1 || (tiles <= groups / n && n * 4 <= steps))
        cost = (float)((tiles * n + 255) / 256) * ((float)((steps + n - 1) / n) + 6.0f) +
               (float)n * ((float)live * (float)hidden / 650000.0f);
    float least = cost;
    for (int d = 32; d; d >>= 1) least = fminf(least, __shfl_xor(least, d));
    return __builtin_ctzll(__builtin_amdgcn_ballot_w64(cost == least)) + 1;
}

// Which tile of D workgroup `id` computes.  Workgroups go round the 8 XCDs;
// each XCD takes a run of consecutive tiles, ordered in bands of 8 columns, so
// that the 32 tiles its CUs work on at a time are 8 x 4 and share operands in
// its L2.
__device__ __forceinline__ void tile_of(int id, int tilesM, int tilesN, int &tm, int &tn)
{
    const int tiles = tilesM * tilesN;
    const int per = tiles / 8, extra = tiles % 8, x = id % 8;
    id = x * per + (x < extra ? x : extra) + id / 8;
    const int band = id / (8 * tilesM), at = id % (8 * tilesM);
    const int width = tilesN - band * 8 < 8 ? tilesN - band * 8 : 8;
    tn = band * 8 + at % width;
    tm = at / width;
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN, int BUFFERS, bool ANY>
struct Product {
    static constexpr int kWaves = WM * WN;
    static constexpr int kThreads = kWaves * 64;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;      // MFMA tiles of a wave
    static constexpr Lie LIE_A = MODE == STATS || MODE == PROB ? ALONG : ACROSS;
    static constexpr Lie LIE_B = MODE == GX ? P_ALONG : MODE == GW ? P_ACROSS : ALONG;
    static constexpr bool A_KC = k_contiguous(LIE_A), B_KC = k_contiguous(LIE_B);
    static constexpr int kStage = (BM + BN) * kStepBytes;
    static constexpr int kLds = BUFFERS * kStage;
    static_assert(!ANY || BUFFERS == 2, "through registers: two halves");
    using LoadA = Loader<T, BM, LIE_A, kWaves>;
    using LoadB = Loader<T, BN, LIE_B, kWaves>;

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

// Beyond this many bytes bf16's gW is stored with the hint that nobody reads it soon: it does not fit the memory's cache
// of 256 MB, and without it what W, X and P have there stays (512 x 4096 x 32768: 509 -> 503 us; 8192 x 4096 x 131072:
// 21.9 -> 21.7 ms).  Below, whoever reads gW next finds it there (with the norm and the clipping behind it, 1024 x
// 2048 x 32768: 520 us, with the hint 528; 1024 x 4096 x 65536: 1900 and 1843 us).  Only whole rows gain: fp32 stores 16
// bytes a lane across rows (256 x 4096 x 32768: 1660 us, with the hint 1690), and the pass for few tokens
// half of a thread's 32 bytes at a time (1 x 4096 x 32768: 205 us, with the hint 334).
constexpr int64_t kPastCaches = (int64_t)1 << 28;

// Writes the staged tile out, whole rows at a time: rows x cols of it.
template <int BM, int THREADS>
__device__ __forceinline__ void write_staged(const unsigned char *lds, bf16_t *to, int64_t ld, int rows, int cols, bool past)
{
    constexpr int kChunks = BM / 8;
    for (int i = threadIdx.x; i < rows * kChunks; i += THREADS) {
        const int row = i / kChunks, col = i % kChunks * 8;
        if (col >= cols) continue;
        const unsigned char *v = lds + staged_at<BM>(row, col);
        bf16_t *p = to + row * ld + col;
        if (col + 8 <= cols) {
            auto *wide = reinterpret_cast<AnyVector<bf16_t>::V *>(p);
            if (past) {
                asm volatile("; past the caches");          // else the compiler joins the two stores and drops the hint
                __builtin_nontemporal_store(*reinterpret_cast<const vint4 *>(v), wide);
                asm volatile("; stored");
            } else {
                *wide = *reinterpret_cast<const vint4 *>(v);
            }
        } else {
            for (int e = 0; e < cols - col; ++e) p[e] = reinterpret_cast<const bf16_t *>(v)[e];
        }
    }
}

// Where element (token n, vocabulary row m) of P lies.
template <typename T> __device__ __forceinline__ int64_t p_byte(int n, int m, int64_t ld)
{
    return n / kBlockTokens * ld + (int64_t)(m / kStep<T>) * kBlockBytes + n % kBlockTokens * kStepBytes +
           m % kStep<T> * (int)sizeof(T);
}

// The tile of gW^T starts from what rounding took from P at the labels: for
// every token whose label is one of the tile's columns, delta times its x.  The
// tokens are found through the groups of 128 vocabulary rows they are sorted by,
// 64 of them at a time (up to 64 tokens are not sorted: every tile looks at all),
// and those of this wave's columns are taken in pairs, so that their rows of x
// are on the way together.  It is done before the first step is asked for: loads come
// back in order, and these would wait for all of it (8192 x 4096 x 131072: 21.7 -> 21.4
// ms; the part that is left, 20 of the 170 us of 1024 x 2048 x 32768, is one in four
// of these multiplications meeting a label).
constexpr int kUnsorted = 64;
template <typename T, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void add_label_remainders(const ProductArgs &g, int m0, int n0, int wm, int wn, int lane,
                                                     int live, vfloat4 (&acc)[BM / WM / 16][BN / WN / 16])
{
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    const int v0 = g.first + n0, v1 = v0 + BN < g.first + g.N ? v0 + BN : g.first + g.N;
    const int from = g.rank ? __builtin_amdgcn_readfirstlane(g.bucket[v0 / 128]) : 0;
    const int to = g.rank ? __builtin_amdgcn_readfirstlane(g.bucket[(v1 + 127) / 128]) : live;
    for (int e0 = from; e0 < to; e0 += 64) {
        const int e = e0 + lane < to ? e0 + lane : to - 1;
        const int2 member = g.rank ? g.member[e] : make_int2(e, g.label[e]);
        const float delta = g.delta[e];
        const int column = member.y - v0;
        unsigned long long mine =
            __builtin_amdgcn_ballot_w64(e0 + lane < to && column >= 0 && column < v1 - v0 && column / (TN * 16) == wn);
        while (mine) {
            int n[2];
            float d[2];
            vint2 x[2][TM];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int at = mine ? __builtin_ctzll(mine) : 0;
                n[p] = __builtin_amdgcn_readlane(column, at) % (TN * 16);
                const float dp = mine ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(delta), at)) : 0.0f;
                d[p] = (lane & 15) == n[p] % 16 ? dp : 0.0f;
                const T *row = reinterpret_cast<const T *>(static_cast<const char *>(g.A) +
                                                           __builtin_amdgcn_readlane(member.x, at) * g.ldA);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const int m = m0 + (wm * TM + i) * 16 + (lane >> 4) * 4;
                    x[p][i] = vint2{0, 0};
                    if (m < g.widthA) x[p][i] = *reinterpret_cast<const vint2 *>(row + m);
                }
                mine &= mine - 1;
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float dj[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) dj[j] = n[p] / 16 == j ? d[p] : 0.0f;
#pragma unroll
                for (int i = 0; i < TM; ++i) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float f = to_float((bf16_t)((unsigned)x[p][i][r >> 1] >> 16 * (r & 1)));
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j][r] = fmaf(dj[j], f, acc[i][j][r]);
                    }
                    __builtin_amdgcn_sched_barrier(0);      // keeps the unpacked values of one row of tiles at a time
                }
            }
        }
    }
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN, int BUFFERS, bool ANY>
__device__ void Product<T, MODE, BM, BN, WM, WN, BUFFERS, ANY>::run(const ProductArgs &g)
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
    const int K = MODE == GW ? (live < g.K ? live : g.K) : g.K;
    const int tilesM = (g.M + BM - 1) / BM, tilesN = (boundN + BN - 1) / BN, tiles = tilesM * tilesN;
    int s0 = 0, s1 = (K + kStep<T> - 1) / kStep<T>, split = 0, id = blockIdx.x;
    if constexpr (MODE == GX) {
        const int splits = splits_of(g.groups, tiles, g.steps, boundN, g.M), steps = s1;
        if (id >= tiles * splits) return;
        split = id / tiles;
        id -= split * tiles;
        s0 = (int)((int64_t)steps * split / splits);
        s1 = (int)((int64_t)steps * (split + 1) / splits);
    } else if (id >= tiles) {
        return;
    }
    int tm, tn;
    tile_of(id, tilesM, tilesN, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;

    LoadA la;
    LoadB lb;
    // ALONG: rows of D's side, of `width` elements; ACROSS: rows of k
    la.template init<(ANY ? 1 : 4)>(g.A, g.ldA, m0, A_KC ? g.M : K, g.widthA, wave, lane);
    lb.template init<(ANY ? 1 : 4)>(g.B, g.ldB, n0, B_KC ? boundN : K, g.widthB, wave, lane);

    vfloat4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    if constexpr (ANY) {
        // Through registers: the next step is on its way while this one is multiplied; several workgroups share a CU.
        const unsigned lane_a = Fragment<T, BM, A_KC>::base(wm * TM * 16, lane);
        const unsigned lane_b = Fragment<T, BN, B_KC>::base(wn * TN * 16, lane) + BM * kStepBytes;
        if (s0 < s1) {
            la.take(s0);
            lb.take(s0);
        }
        for (int s = s0; s < s1; ++s) {
            const unsigned half = ((s - s0) & 1) * kStage;
            la.put(lds_raw + half, wave, lane);
            lb.put(lds_raw + half + BM * kStepBytes, wave, lane);
            __syncthreads();        // also: nobody reads the other half any more
            if (s + 1 < s1) {
                la.take(s + 1);
                lb.take(s + 1);
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                vint4 b[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) b[j] = Fragment<T, BN, B_KC>::read(lds, lane_b + half, j, kk);
                vint4 valid = {-1, -1, -1, -1};
                if (LIE_A == ALONG && s + 1 == s1) valid = valid_k<T>(K - s * kStep<T> - (4 * kk + (lane >> 4)) * (16 / (int)sizeof(T)));
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    multiply<T>(Fragment<T, BM, A_KC>::read(lds, lane_a + half, i, kk) & valid, b, acc[i]);
            }
        }
    } else
    // BUFFERS tiles in LDS, a step each; a step is two halves of k, and the TM
    // rows of MFMA tiles of one half are a group each.  The fragment of A is read
    // three groups ahead into a ring of four, those of B for one half of k while
    // the other half is multiplied.  The step changes three groups before its
    // end: all its fragments are in registers by then, so the tile just read can
    // be refilled, and the matrix cores have work while the waves meet and the
    // next step's first fragments come out of LDS.
    if (s0 < s1) {
        constexpr int RING = 4, AHEAD = 3, GROUPS = 2 * TM, LAST = GROUPS - AHEAD, SPREAD = TM < LAST ? TM : LAST;
        static_assert(GROUPS % RING == 0, "the ring closes with the step");
        vint4 a[RING], b[2][TN];
        using FragmentA = Fragment<T, BM, A_KC>;
        using FragmentB = Fragment<T, BN, B_KC>;
        const unsigned lane_a = FragmentA::base(wm * TM * 16, lane);
        const unsigned lane_b = FragmentB::base(wn * TN * 16, lane) + BM * kStepBytes;
        unsigned at_a = lane_a, at_b = lane_b;
        // the half that is read from now on; the addresses of single fragments are made where they are used (kept in
        // registers they would not fit)
        auto read_from = [&](unsigned half) {
            at_a = lane_a + half;
            at_b = lane_b + half;
            asm("" : "+v"(at_a), "+v"(at_b));
        };
        auto read_a = [&](int group) { a[group % RING] = FragmentA::read(lds, at_a, group % TM, group / TM); };
        auto read_b = [&](int kk, int j) { b[kk][j] = FragmentB::read(lds, at_b, j, kk); };
        vint4 ra, rb;
        unsigned ka[2], kb[2], to = 0;
        constexpr int kCalls = LoadA::kCalls + LoadB::kCalls;
        auto aim = [&](int s, unsigned at) {
            la.aim(s, s1, ra, ka);
            lb.aim(s, s1, rb, kb);
            to = lds0 + at;
        };
        auto call = [&](int c) {
            if (c < LoadA::kCalls) la.call(c, ra, ka, to, wave);
            else lb.call(c - LoadA::kCalls, rb, kb, to + BM * kStepBytes, wave);
        };
        // In the last step a chunk of a row of A may run past the row's end, into whatever follows it.
        vint4 valid[2];
        auto group = [&](int g, bool last) {
            vint4 x = a[g % RING];
            if (LIE_A == ALONG && last) x &= valid[g / TM];
            multiply<T>(x, b[g / TM], acc[g % TM]);
        };
        // Steps past the end are asked for too where more than two tiles are open (they bring zeros), so that what
        // is open is the same number of calls in every step.
        constexpr int kOpen = (BUFFERS - 2) * kCalls;
        if constexpr (MODE == GW && sizeof(T) == 2)
            add_label_remainders<T, BM, BN, WM, WN>(g, m0, n0, wm, wn, lane, live, acc);
        aim(s0, 0);
#pragma unroll
        for (int c = 0; c < kCalls; ++c) call(c);
#pragma unroll
        for (int x = 1; x + 1 < BUFFERS; ++x) {
            aim(s0 + x, x * kStage);
#pragma unroll
            for (int c = 0; c < kCalls; ++c) call(c);
        }
        wait_and_meet<kOpen>();
        if (BUFFERS > 2 || s0 + 1 < s1) {
            aim(s0 + BUFFERS - 1, (BUFFERS - 1) * kStage);
#pragma unroll
            for (int c = 0; c < kCalls; ++c) call(c);
        }
        unsigned now = 0;
#pragma unroll
        for (int j = 0; j < TN; ++j) read_b(0, j);
#pragma unroll
        for (int g = 0; g < AHEAD; ++g) read_a(g);
        auto most = [&](bool last) {
#pragma unroll
            for (int g = 0; g < LAST; ++g) {
                read_a(g + AHEAD);
                if (g < SPREAD) {
#pragma unroll
                    for (int j = TN * g / SPREAD; j < TN * (g + 1) / SPREAD; ++j) read_b(1, j);
                }
                group(g, last);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (int s = s0; s + 1 < s1; ++s) {
            most(false);
            wait_and_meet<kOpen>();
            const bool more = BUFFERS > 2 || s + 2 < s1;
            if (more) aim(s + BUFFERS, now);
            now = now + kStage == kLds ? 0 : now + kStage;
            read_from(now);
#pragma unroll
            for (int g = LAST; g < GROUPS; ++g) {
                const int x = g - LAST;
#pragma unroll
                for (int j = TN * x / AHEAD; j < TN * (x + 1) / AHEAD; ++j) read_b(0, j);
                read_a(x);
                group(g, false);
                if (more) {
#pragma unroll
                    for (int c = kCalls * x / AHEAD; c < kCalls * (x + 1) / AHEAD; ++c) call(c);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (LIE_A == ALONG) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                valid[kk] = valid_k<T>(K - (s1 - 1) * kStep<T> - (4 * kk + (lane >> 4)) * (16 / (int)sizeof(T)));
            }
        }
        most(true);
#pragma unroll
        for (int g = LAST; g < GROUPS; ++g) group(g, true);
        if constexpr (BUFFERS > 2) wait_and_meet();         // nothing may be on its way into LDS when the workgroup ends
    }

    const int mw = m0 + wm * TM * 16 + (lane >> 4) * 4, nw = n0 + wn * TN * 16 + (lane & 15);
    const int m_wave = m0 + wm * TM * 16;
    if constexpr (MODE == STATS) {
        wait_and_meet();
        float2 *red = reinterpret_cast<float2 *>(lds_raw);      // [wm][column]
        const float scale = scale_of<T>(g.alpha);
        const bool tail = m0 + BM > g.M;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 16;
            const int want = n < boundN ? g.label[n] - g.first : -1;
            // the label's logit: few tiles hold one
            if (__builtin_amdgcn_ballot_w64(want >= m_wave && want < m_wave + TM * 16 && want < g.M)) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (mw + i * 16 + r == want && want < g.M) g.target[n] = g.alpha * acc[i][j][r];
            }
            float top = -INFINITY, sum = 0.0f;
            if (!tail && g.alpha > 0.0f) {
                // the maximum of the products is that of the logits
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum += exponential<T>((acc[i][j][r] - from) * scale);
                top *= g.alpha;
            } else {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (mw + i * 16 + r < g.M) top = fmaxf(top, g.alpha * acc[i][j][r]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (mw + i * 16 + r < g.M)
                            sum += exponential<T>((g.alpha * acc[i][j][r] - from) * scale_of<T>(1.0f));
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 16) red[wm * BN + (wn * TN + j) * 16 + lane] = make_float2(top, sum);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BN; c += kThreads) {
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WM; ++w) top = fmaxf(top, red[w * BN + c].x);
            const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < WM; ++w) sum += red[w * BN + c].y * expf(red[w * BN + c].x - from);
            if (n0 + c < boundN) g.stats[(int64_t)tm * g.ldStats + n0 + c] = make_float2(top, sum);
        }
    } else if constexpr (MODE == PROB) {
        // P is rounded to the operands' type, since the two products that follow run on it: each element is off
        // by at most half a step of that type (bf16: 2^-8 of itself), and the sums over tokens or vocabulary
        // average that out - except at the label, whose element mostly outweighs the others: what its rounding
        // took is kept (bf16) and goes into both products in fp32.  Elsewhere it stays: a row of gW that is
        // nobody's label, and a token whose softmax lies on another row than its label's, have it on top of the
        // result's own rounding.  Past the last token and the last vocabulary row the tile is zeros, which the
        // products may run into.
        unsigned char *P = static_cast<unsigned char *>(g.P);
        const float scale = scale_of<T>(g.alpha);
        const bool tail = m0 + BM > g.M;
        if constexpr (sizeof(T) == 2) wait_and_meet();
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 16;
            const bool live_n = n < boundN;
            const float lse = live_n ? g.lse[n] * scale_of<T>(1.0f) : 0.0f, both = live_n ? g.both[n] : 0.0f;
            const int want = live_n ? g.label[n] - g.first : -1;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = exponential<T>(fmaf(acc[i][j][r], scale, -lse)) * both;
            if (__builtin_amdgcn_ballot_w64(want >= m_wave && want < m_wave + TM * 16)) {
                const float gloss = live_n ? g.gloss[n] : 0.0f;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (mw + i * 16 + r == want) {
                            const float p = acc[i][j][r] - gloss;
                            acc[i][j][r] = p;
                            if constexpr (sizeof(T) == 2) g.delta[g.rank ? g.rank[n] : n] = p - to_float(from_float<T>(p));
                        }
            }
            if (tail || n0 + BN > boundN) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!live_n || mw + i * 16 + r >= g.M) acc[i][j][r] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = mw + i * 16;
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = from_float<T>(acc[i][j][r]);
                if constexpr (sizeof(T) == 2) {
                    *reinterpret_cast<vint2 *>(lds_raw + staged_at<BM>(n - n0, m - m0)) = *reinterpret_cast<vint2 *>(v);
                } else {
                    *reinterpret_cast<vint4 *>(P + p_byte<T>(n, m, g.ldP)) = *reinterpret_cast<vint4 *>(v);
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            __syncthreads();
            // along the rows of a block, block by block; GW takes rows in steps, which a narrow tile does not fill
            constexpr int kRows = BN < kStep<T> ? kStep<T> : BN;
            for (int i = threadIdx.x; i < kRows * (BM / 8); i += kThreads) {
                const int row = i / 8 % kRows, col = i / 8 / kRows * kStep<T> + i % 8 * 8;
                vint4 v = {0, 0, 0, 0};
                if (row < BN) v = *reinterpret_cast<const vint4 *>(lds_raw + staged_at<BM>(row, col));
                *reinterpret_cast<vint4 *>(P + p_byte<T>(n0 + row, m0 + col, g.ldP)) = v;
            }
        }
    } else if constexpr (MODE == GX) {
        float *part = g.part + (int64_t)split * boundN * g.ldD;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nw + j * 16;
            if (n >= boundN) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = mw + i * 16;
                if (m >= g.M) continue;         // ldD is a multiple of 4: four fit where one does
                vfloat4 *to = reinterpret_cast<vfloat4 *>(part + (int64_t)n * g.ldD + m);
                vfloat4 v = acc[i][j];
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
            const int n = nw + j * 16;
            if (n >= boundN) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = mw + i * 16;
                T *to = out + (int64_t)n * g.ldD + m;
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = acc[i][j][r];
                    if (g.beta != 0.0f && m + r < g.M) x += g.beta * to_float(to[r]);
                    v[r] = from_float<T>(x);
                }
                if constexpr (sizeof(T) == 2) {
                    *reinterpret_cast<vint2 *>(lds_raw + staged_at<BM>(n - n0, m - m0)) = *reinterpret_cast<vint2 *>(v);
                } else if (m + 4 <= g.M) {
                    *reinterpret_cast<AnyVector<float>::V *>(to) = *reinterpret_cast<vint4 *>(v);
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
                                       g.M - m0 < BM ? g.M - m0 : BM, g.past);
        }
    }
}

template <typename T, Mode MODE, int BM, int BN, int WM, int WN, int BUFFERS, bool ANY>
__global__ void __launch_bounds__(WM *WN * 64, MODE == GW && WM * WN == 4 ? 3 : 2)
product_kernel(ProductArgs g)
{
    Product<T, MODE, BM, BN, WM, WN, BUFFERS, ANY>::run(g);
}

}  // namespace xent
}  // namespace ulmgpu
#endif
