// Shared pieces of the sequence operators (rotary.hip, attn_window.hip, attn_window_step.hip): element types, ragged
// sequences, the window + sinks rule.
#pragma once
#include "common.hip.h"

namespace qcn_seq {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kMaxDim = 128;

template <class T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }
// one rounding to nearest even at the store; everything before it is fp32
template <class T> __device__ __forceinline__ T from_f32(float x) { return (T)x; }

static inline size_t dtype_bytes(int64_t dtype) { return dtype == QCN_DTYPE_F32 ? 4 : 2; }
static inline bool dtype_known(int64_t dtype) { return dtype == QCN_DTYPE_F32 || dtype == QCN_DTYPE_F16 || dtype == QCN_DTYPE_BF16; }

// a strided row tensor [tokens, heads, dim]: the features of a head are contiguous
struct Rows {
    int64_t tok, head;   // strides in elements
};

constexpr int64_t kMaxHeads = 32767;            // of one tensor
// a launch counts its threads in 32 bits, and the blocks here have 256
constexpr int64_t kMaxBlocks = ((int64_t)1 << 24) - 1;
constexpr int64_t kMaxTokStride = (int64_t)1 << 24;   // elements: 64 rows' offsets are 32-bit

// rows are loaded in 16-byte pieces, and strides do not point backwards
static inline bool rows_aligned(const void *p, int64_t tok, int64_t head, int64_t dtype)
{
    const int64_t piece = 16 / (int64_t)dtype_bytes(dtype);
    return ((uintptr_t)p & 15) == 0 && tok >= 0 && head >= 0 && tok % piece == 0 && head % piece == 0;
}

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : (x > hi ? hi : x); }

// Boundaries of sequence b, forced into [0, n]: a boundary tensor that is wrong on the device gives wrong rows but no access
// outside the token tensors.
__device__ __forceinline__ void seq_range(const int64_t *__restrict__ cu, int64_t b, int64_t n, int64_t &beg, int64_t &end)
{
    beg = clamp64(cu[b], 0, n);
    end = clamp64(cu[b + 1], beg, n);
}

// Ragged tiles without a host round trip: sequence b owns the tile numbers  start(b) .. start(b + 1) - 1  with
// start(b) = (cu[b] * rows >> shift) + b, tiles of 2^shift rows.  That is at least ceil(len * rows / tile) numbers for every
// sequence (the floor of a sum is at least the sum of the floors), at most one too many, and start() needs no prefix sum.
// Number n_seq stands for the rows behind the last sequence.
//
// The wave looks for the last b in [0, n_seq] with start(b) <= tile, 64 candidates at a time: first around where b would be if
// all sequences were of one length (mostly right, so one dependent load), else by narrowing 64-fold.  The boundaries of b come
// with the last look: beg = cu[b], end = cu[b + 1] (n for n_seq), forced into range as in seq_range.
struct Found {
    int64_t b, beg, end;
};
__device__ __forceinline__ int64_t wave_get(int64_t v, int lane)
{
    const unsigned lo = __builtin_amdgcn_readlane((int)(v & 0xffffffff), lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ Found find_seq(const int64_t *__restrict__ cu, int64_t n_seq, int64_t n, int64_t rows, int shift, int64_t tile,
                                          int64_t n_tiles, int lane)
{
    int64_t lo = 0, count = n_seq + 1;   // candidates lo .. lo + count - 1
    int64_t base = 0, value = 0;
    uint64_t hits = 0;
    const auto look = [&](int64_t from) {
        const int64_t c = from + lane < n_seq ? from + lane : n_seq;
        base = from;
        value = clamp64(cu[c], 0, n);
        hits = __ballot(from + lane < lo + count && (value * rows >> shift) + c <= tile);
    };
    bool found = false;
    if (count > 64) {
        int64_t guess = (int64_t)((float)tile * ((float)n_seq / (float)n_tiles)) - 31;
        guess = clamp64(guess, 0, n_seq - 63);
        look(guess);
        if (!(hits & 1) && guess > 0) count = guess;                              // it lies in front
        else if (hits == ~0ull && guess + 64 <= n_seq) { lo = guess + 63; count = n_seq + 1 - lo; }   // or behind
        else found = true;
        while (!found && count > 64) {
            const int64_t step = (count + 63) / 64, b = lo + (int64_t)lane * step;
            const bool in = (int64_t)lane * step < count;
            const bool ok = in && (clamp64(cu[in ? b : lo], 0, n) * rows >> shift) + b <= tile;
            const int last = 63 - __builtin_clzll(__ballot(ok) | 1ull);
            const int64_t next = lo + (int64_t)last * step, left = lo + count - next;
            lo = next;
            count = left < step ? left : step;
        }
    }
    if (!found) look(lo);
    const int last = 63 - __builtin_clzll(hits | 1ull);
    Found f;
    f.b = base + last;
    f.beg = wave_get(value, last);
    f.end = f.b >= n_seq ? n : (last < 63 ? wave_get(value, last + 1) : clamp64(cu[f.b + 1], 0, n));
    if (f.end < f.beg) f.end = f.beg;
    return f;
}

// slot of position p in a cache of `sinks` first tokens and a ring of `window`
__device__ __forceinline__ int64_t cache_slot(int64_t p, int64_t sinks, int64_t window)
{
    return p < sinks ? p : sinks + (p - sinks) % window;
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Values that are not finite, as numbers that a product can count: +inf 1, -inf 128, NaN both.  The products of the codes of up to
// 127 keys with 1 (a row sees the key) or 0 say what the row's sum holds of each.
__device__ __forceinline__ float value_code(float v)
{
    return fabsf(v) < INFINITY ? 0.f : (v > 0.f ? 1.f : (v < 0.f ? 128.f : 129.f));
}
__device__ __forceinline__ float counted_sum(float c)   // +inf, -inf, NaN (of both) or 0
{
    const float minus = floorf(c * (1.f / 128.f));
    return (c > 128.f * minus ? INFINITY : 0.f) + (minus > 0.f ? -INFINITY : 0.f);
}

// ---------------------------------------------------------------------------------------------------------------------
// matrix operands
// ---------------------------------------------------------------------------------------------------------------------
// Both attention kernels form S^T = K Q^T and O^T = V^T P^T.  A lane of the accumulator then holds ONE query (column) and some
// keys (rows), so softmax statistics are per lane plus one or two lane exchanges, and the accumulator of S^T is, register for
// register, the B operand of the second product: the order of the contraction index is free as long as V^T follows it.
//   32 x 32 accumulator:  column = lane & 31, row = (r & 3) + 8 (r >> 2) + 4 (lane >> 5)
//   16 x 16 accumulator:  column = lane & 15, row = r + 4 (lane >> 4)
template <class T> struct Mat;
template <> struct Mat<_Float16> {
    using V8 = f16x8;
    using V4 = __attribute__((ext_vector_type(4))) _Float16;
    static __device__ __forceinline__ f32x16 mul32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    // c + x[2 i] + x[2 i + 1], products with 1 in fp32
    static __device__ __forceinline__ float add_pair(V8 x, int i, float c)
    {
        using V2 = __attribute__((ext_vector_type(2))) _Float16;
        return __builtin_amdgcn_fdot2(V2{x[2 * i], x[2 * i + 1]}, V2{(_Float16)1.f, (_Float16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 mul16(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mul16(V4 a, V4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<__bf16> {
    using V8 = bf16x8;
    using V4 = __attribute__((ext_vector_type(4))) __bf16;
    using S4 = __attribute__((ext_vector_type(4))) short;
    static __device__ __forceinline__ f32x16 mul32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float add_pair(V8 x, int i, float c)
    {
        using V2 = __attribute__((ext_vector_type(2))) __bf16;
        return __builtin_amdgcn_fdot2_f32_bf16(V2{x[2 * i], x[2 * i + 1]}, V2{(__bf16)1.f, (__bf16)1.f}, c, false);
    }
    static __device__ __forceinline__ f32x4 mul16(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mul16(V4 a, V4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(S4, a), __builtin_bit_cast(S4, b), c, 0, 0, 0);
    }
};

// ds_read_b64_tr_b16: the 16 lanes of a group read 8 bytes each, taken as 4 rows (lanes 4 j .. 4 j + 3) of 16 elements; lane l
// gets column l: element j from row j.  (Checked lane by lane on the card.)
__device__ __forceinline__ uint2 lds_read_transposed(const void *p)
{
    using S4 = __attribute__((ext_vector_type(4))) short;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4 *)p));
}

// Largest and sum over lanes l, l ^ 32 (halves), and over l, l ^ 16, l ^ 32, l ^ 48 (quarters).  v_permlane32_swap of a value with
// itself leaves the low half's value in all lanes of one result and the high half's in the other; v_permlane16_swap likewise
// for the 16-lane rows of each half.
struct Pair { float a, b; };
__device__ __forceinline__ Pair both_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned x = r[0], y = r[1];   // (a bit cast of a vector's element in place takes its first element)
    return {__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ Pair both_rows(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned x = r[0], y = r[1];   // (a bit cast of a vector's element in place takes its first element)
    return {__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)};
}
__device__ __forceinline__ float halves_max(float v) { const Pair p = both_halves(v); return fmaxf(p.a, p.b); }
__device__ __forceinline__ float halves_sum(float v) { const Pair p = both_halves(v); return p.a + p.b; }
__device__ __forceinline__ float quarters_max(float v) { const Pair p = both_rows(halves_max(v)); return fmaxf(p.a, p.b); }
__device__ __forceinline__ float quarters_sum(float v) { const Pair p = both_rows(halves_sum(v)); return p.a + p.b; }

// 1 / sum of a softmax whose largest term is at least 1 (the running maximum is at most the largest score), 0 for an empty row
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kMaxScale = 2.35e38;   // times log2(e) it is still a float: an infinite one would make NaN of a score of 0

}  // namespace qcn_seq
