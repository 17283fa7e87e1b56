// The serving form of attn_window.hip: a cache of `sinks` first tokens and a ring of the last `window`, per sequence.
//
// Position p lives in slot p (p < sinks) or sinks + (p - sinks) mod window.  When position p has been written, the filled slots
// are the first min(p + 1, sinks + window), and they hold exactly the positions p may see: [0, sinks) and (p - window, p]
// (while p < sinks + window nothing has been overwritten and the window reaches down to the sinks).  Softmax does not depend
// on the order of its terms, so a step reads the slots as they lie.
//
// Caches are [batch, kv heads, sinks + window, dim]: the keys of one head are one contiguous stretch.
#include "sequence.hip.h"

namespace {

using namespace qcn_seq;

constexpr int kAppendShift = 4;   // tokens of a block: 16
constexpr int64_t kMaxLength = (int64_t)1 << 62;   // a length above it is no length: positions behind it stay in 64 bits

struct AppendArgs {
    const void *k, *v;
    Rows kr, vr;
    const int64_t *cu, *lengths;
    const uint8_t *key_mask;
    int64_t n_seq, n;
    int hk, dim, pieces;          // 16-byte pieces of a head row
    int64_t window, sinks, slots;
    void *k_cache, *v_cache;
    uint8_t *mask_cache;
};

// A block takes 16 tokens of one sequence; a thread moves one 16-byte piece of k and of v.  A token that a later one of the
// same call would overwrite is not moved, so every slot has one writer.
// Bound by memory: 1600 x 59 tokens x 8 heads of 16 in float32 (167 MB read and written) 35.7 us, 4.7 TB/s, what a library copy
// reaches; ragged prompts of up to 2500 tokens x 8 heads of 128 into windows of 1024 (104 MB) 23.5 us.  Heads next to each other moved
// together for whole cache lines, blocks of 32 tokens, and four pieces of a thread in flight were no faster (36.9, 39, 37 us).
template <class T>
__global__ __launch_bounds__(256) void window_cache_append_kernel(AppendArgs a)
{
    const Found f = find_seq(a.cu, a.n_seq, a.n, 1, kAppendShift, blockIdx.x, gridDim.x, threadIdx.x & 63);
    if (f.b == a.n_seq) return;                             // behind the last sequence: left as they are
    const int64_t b = f.b, beg = f.beg, end = f.end;
    const int64_t first = ((int64_t)blockIdx.x - ((beg >> kAppendShift) + b)) << kAppendShift;
    const int64_t old = a.lengths[b];
    if (first < 0 || first >= end - beg || old < 0 || old > kMaxLength) return;
    const int64_t total = old + (end - beg);
    const int64_t ntok = end - beg - first < (1 << kAppendShift) ? end - beg - first : (1 << kAppendShift);
    // nothing of the tile stays (the sinks are the first positions, the window the last)
    if (old + first >= a.sinks && old + first + ntok <= total - a.window) return;
    constexpr int kPiece = 16 / (int)sizeof(T);
    const int per_head = (int)ntok * a.pieces;
    for (int i = threadIdx.x; i < per_head * a.hk; i += 256) {
        const int h = i / per_head, r = i % per_head;
        const int64_t t = first + r / a.pieces;
        const int d = (r % a.pieces) * kPiece;
        const int64_t p = old + t;
        if (p >= a.sinks && p < total - a.window) continue;
        const int64_t slot = cache_slot(p, a.sinks, a.window);
        const u32x4 kv = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const T *>(a.k) + (beg + t) * a.kr.tok + h * a.kr.head + d);
        const u32x4 vv = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const T *>(a.v) + (beg + t) * a.vr.tok + h * a.vr.head + d);
        const int64_t to = ((b * a.hk + h) * a.slots + slot) * a.dim + d;
        *reinterpret_cast<u32x4 *>(reinterpret_cast<T *>(a.k_cache) + to) = kv;
        *reinterpret_cast<u32x4 *>(reinterpret_cast<T *>(a.v_cache) + to) = vv;
        if (a.mask_cache && h == 0 && d == 0) a.mask_cache[b * a.slots + slot] = a.key_mask ? (a.key_mask[beg + t] != 0) : 1;
    }
}

struct StepArgs {
    const void *q, *k, *v;
    Rows qr, kr, vr;
    const int64_t *lengths;
    const uint8_t *key_mask;
    int64_t batch;
    int hq, hk, group, dim;
    int64_t window, sinks, slots;
    float c2;                     // scale in base 2
    void *k_cache, *v_cache;
    uint8_t *mask_cache;
    void *out;                    // [batch, hq, dim] contiguous
};

// A task is a cache row, a key head, up to 16 of the query heads that share it, and a part of the filled slots.  Its waves take
// chunks of 32 or 64 slots in turn:  S^T (slots x heads) = K Q^T, O^T (features x heads) = V^T P^T with 16 x 16 accumulators, so that a
// shared key head is read once for its whole group.
//
// HBM-bound: every filled slot is read once.  K goes straight into registers as the A operand (a lane reads 16 bytes of a slot,
// four lanes 64).  V has to be transposed: 16-bit rows pass through LDS that belongs to the wave alone (no barrier) and come
// back by transposing reads.  Of float32 a lane reads the features it multiplies: straight from memory where a row is 256 bytes or
// more, through LDS where that would be loads of 4 or 8 bytes.
// The new token is read from the inputs, never from its slot, which another block of this launch is writing.
//
// Weights meet 16-bit V in two products: rounded to its type, and with what that rounding left (16 bits of bfloat16, 22 of float16
// together), so the output's rounding is the only one to 16 bits.  The kernel waits for memory, and that hardly shows where it has much to
// read (us, one product and two, with the look for values that are not finite that the second needs): 64 x 8 key heads x 4100 slots 170 and
// 171, one request 19.9 and 20.4, 256 x 4 heads of 64 x 1004 slots 47.8 and 48.5, 64 x 8 x 240 slots 25.1 and 26.6, 1600 agents x 8 x 51
// slots in bfloat16 19.2 and 20.2.
// Measured: that step (64 requests x 32 heads of 128 in bfloat16) 169.7 us, 984 MB at 5.8 TB/s; one request 10.4 + 4.7 us (two launches,
// three memory latencies each); 1600 agents x 8 heads of 16 x 51 slots in float32 21.9 us, 3.6 TB/s.
template <class T, int DP> struct Step {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NU = DP <= 32 ? 4 : 2, CHUNK = 16 * NU;                        // slots of a chunk: narrow heads take 64
    static constexpr int VW = !F32 ? 1 : (DP % 64 == 0 ? 4 : (DP % 32 == 0 ? 2 : 1));   // float32: features of a lane's V load
    static constexpr int SB = 16 * VW, NSB = DP / SB;
    static constexpr bool TURN = !F32 || DP <= 32;         // V passes through LDS
    static constexpr int PIECES = DP * (int)sizeof(T) / 16, PIECE = 16 / (int)sizeof(T);   // 16-byte pieces of a row, elements of one
    static constexpr int O_STRIDE = DP + 4;               // floats: a row's pad keeps 16 heads off one bank
    static constexpr int V_ROW = F32 ? O_STRIDE * 4 : DP * 2;                           // bytes of a V row in LDS
    static constexpr int V_BYTES = TURN ? CHUNK * V_ROW : 0, O_BYTES = 64 * O_STRIDE;   // a chunk of V, then 16 rows of O
    static constexpr int WAVE_BYTES = V_BYTES > O_BYTES ? V_BYTES : O_BYTES;
};

// 8 rows x 32 bytes of a transposing read (half a wave) cover all banks
template <int DP> __device__ __forceinline__ int v_piece(int row, int piece)
{
    return piece ^ (DP == 128 ? (row & 7) << 1 : DP == 64 ? ((row >> 1) & 3) << 1 : DP == 16 ? 0 : ((row >> 2) & 1) << 1);
}

template <class T, int N> struct alignas(sizeof(T) * N) Pack { T e[N]; };

struct Part {
    int heads, head0, kvh;    // query heads of the task
    int64_t b, p, slot, n;    // cache row, position of the new token and its slot, filled slots
    int64_t c0, c1;           // slots of this task
};

template <class T, int DP>
__device__ __forceinline__ void attend_slots(const StepArgs &a, const Part &t, int wave, int waves, int lane, char *lds,
                                             f32x4 (&o)[DP / 16], float &m, float &l)
{
    using L = Step<T, DP>;
    const int n = lane & 15, g = lane >> 4;
    const int head = t.head0 + (n < t.heads ? n : t.heads - 1);
    const T *q = reinterpret_cast<const T *>(a.q) + t.b * a.qr.tok + head * a.qr.head;
    const T *kn = reinterpret_cast<const T *>(a.k) + t.b * a.kr.tok + t.kvh * a.kr.head;
    const T *vn = reinterpret_cast<const T *>(a.v) + t.b * a.vr.tok + t.kvh * a.vr.head;
    const int64_t base = (t.b * a.hk + t.kvh) * a.slots * a.dim;
    const T *kc = reinterpret_cast<const T *>(a.k_cache) + base, *vc = reinterpret_cast<const T *>(a.v_cache) + base;
    const uint8_t *mask = a.mask_cache ? a.mask_cache + t.b * a.slots : nullptr;
    const bool new_seen = !mask || !a.key_mask || a.key_mask[t.b] != 0;

    constexpr int NQ = L::F32 ? DP / 16 : (DP + 31) / 32;
    u32x4 qf[NQ];
    const auto piece = [&](const T *row, int d) {          // 16 bytes of a row's features, zero past its end
        u32x4 x = *reinterpret_cast<const u32x4 *>(row + (d < a.dim ? d : 0));
        if (d >= a.dim) x = u32x4{0, 0, 0, 0};
        return x;
    };
#pragma unroll
    for (int c = 0; c < NQ; ++c) qf[c] = piece(q, L::F32 ? 16 * c + 4 * g : 32 * c + 8 * g);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;

    for (int64_t j0 = t.c0 + L::CHUNK * wave; j0 < t.c1; j0 += L::CHUNK * waves) {
        const auto row_of = [&](const T *cache, const T *fresh, int r) {
            int64_t c = j0 + r;
            c = c < t.c1 ? c : t.c1 - 1;
            return c == t.slot ? fresh : cache + c * a.dim;
        };
        u32x4 kf[L::NU][NQ];
#pragma unroll
        for (int u = 0; u < L::NU; ++u) {
            const T *row = row_of(kc, kn, 16 * u + n);
#pragma unroll
            for (int c = 0; c < NQ; ++c) kf[u][c] = piece(row, L::F32 ? 16 * c + 4 * g : 32 * c + 8 * g);
        }
        const int64_t cl = j0 + lane;
        const bool in = lane < L::CHUNK && cl < t.c1;
        const bool ok = in && (cl == t.slot ? new_seen : (!mask || mask[in ? cl : t.c1 - 1] != 0));
        constexpr int NV = L::TURN ? (L::CHUNK * L::PIECES + 63) / 64 : 1;
        u32x4 vf[NV];
        using PV = Pack<T, L::VW>;
        if constexpr (L::TURN) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int x = lane + 64 * i, r = x / L::PIECES;
                vf[i] = piece(row_of(vc, vn, r), x % L::PIECES * L::PIECE);
            }
        }
        const uint64_t seen = __ballot(ok);
        f32x4 s[L::NU];
#pragma unroll
        for (int u = 0; u < L::NU; ++u) {
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NQ; ++c) {
                if constexpr (L::F32) {
                    const f32x4 kk = __builtin_bit_cast(f32x4, kf[u][c]), qq = __builtin_bit_cast(f32x4, qf[c]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], qq[e], s[u], 0, 0, 0);
                } else {
                    using V8 = typename Mat<T>::V8;
                    s[u] = Mat<T>::mul16(__builtin_bit_cast(V8, kf[u][c]), __builtin_bit_cast(V8, qf[c]), s[u]);
                }
            }
        }
        if constexpr (L::TURN) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int x = lane + 64 * i, r = x / L::PIECES, c = x % L::PIECES;
                // 0 times what a masked slot holds must stay 0
                const u32x4 v = (seen >> r) & 1 ? vf[i] : u32x4{0, 0, 0, 0};
                *reinterpret_cast<u32x4 *>(lds + r * L::V_ROW + (L::F32 ? c : v_piece<DP>(r, c)) * 16) = v;
            }
            // the wave's own LDS: these writes are done in order before the reads below; only the compiler is to keep them apart
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < L::NU; ++u) {
            const unsigned w = (unsigned)(seen >> (16 * u)) >> (4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (!((w >> r) & 1)) s[u][r] = -INFINITY;
                top = fmaxf(top, s[u][r]);
            }
        }
        top = quarters_max(top);
        // the maximum follows only jumps of more than 2^8: until then p stays below 2^8 and nothing is rescaled
        const float scaled = top * a.c2;
        if (__ballot(scaled > m + 8.f)) {
            const float mn = scaled > m ? scaled : m;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) o[i] *= alpha;
            m = mn;
        }
        const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int u = 0; u < L::NU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], a.c2, -at));
                l += s[u][r];
            }
        if constexpr (L::F32) {
#pragma unroll
            for (int u = 0; u < L::NU; ++u) {
                const unsigned w = (unsigned)(seen >> (16 * u)) >> (4 * g);
#pragma unroll
                for (int sb = 0; sb < L::NSB; ++sb) {
                    PV v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = sb * L::SB + L::VW * n, c = 16 * u + 4 * g + r;
                        if constexpr (L::TURN) {
                            v[r] = *reinterpret_cast<const PV *>(lds + c * L::V_ROW + d * (int)sizeof(T));
                        } else {
                            v[r] = *reinterpret_cast<const PV *>(row_of(vc, vn, c) + (d < a.dim ? d : 0));
                            if (!((w >> r) & 1)) v[r] = PV{};
                        }
                    }
#pragma unroll
                    for (int e = 0; e < L::VW; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            o[sb * L::VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r].e[e], s[u][r], o[sb * L::VW + e], 0, 0, 0);
                }
            }
        } else {
            using V8 = typename Mat<T>::V8;
#pragma unroll
            for (int half = 0; half < L::NU / 2; ++half) {
                V8 hi, lo;                                     // p = hi + lo
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = s[2 * half + (i >> 2)][i & 3];
                    hi[i] = from_f32<T>(p);
                    lo[i] = from_f32<T>(p - to_f32(hi[i]));
                }
                const int i16 = lane & 15, r = 32 * half + 4 * g + (i16 >> 2);
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) {
                    const int c = 2 * dt + ((i16 >> 1) & 1), byte = 8 * (i16 & 1);
                    const uint2 x = lds_read_transposed(lds + r * L::V_ROW + v_piece<DP>(r, c) * 16 + byte);
                    const uint2 y = lds_read_transposed(lds + (r + 16) * L::V_ROW + v_piece<DP>(r + 16, c) * 16 + byte);
                    const V8 vt = __builtin_bit_cast(V8, u32x4{x.x, x.y, y.x, y.y});
                    o[dt] = Mat<T>::mul16(vt, hi, o[dt]);
                    o[dt] = Mat<T>::mul16(vt, lo, o[dt]);
                }
            }
        }
        if constexpr (L::TURN) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if constexpr (!L::F32) {
        // An infinite value has met two parts of a weight, of which one may be 0 or below.  All heads of the task see the same slots, so
        // the values alone say what becomes of such a feature: they are gone over again, without keys and weights, 32 slots at a time.
        f32x4 any = o[0];                                  // not finite if an element is not (an overflow costs a look)
#pragma unroll
        for (int i = 1; i < DP / 16; ++i) any += o[i];
        const float sum = (any[0] + any[1]) + (any[2] + any[3]);
        if (__ballot(!(fabsf(sum) < INFINITY) && l == l)) {
            using V8 = typename Mat<T>::V8;
            V8 one;
#pragma unroll
            for (int i = 0; i < 8; ++i) one[i] = (T)1.f;
            f32x4 held[DP / 16];                           // 0, or what is not finite among a feature's values
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) held[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int64_t j0 = t.c0 + 32 * wave; j0 < t.c1; j0 += 32 * waves) {
#pragma unroll 1
                for (int x = lane; x < 32 * L::PIECES; x += 64) {
                    const int r = x / L::PIECES, c = x % L::PIECES;
                    const int64_t slot = j0 + r;
                    u32x4 v = {0, 0, 0, 0};
                    if (slot < t.c1 && (slot == t.slot ? new_seen : (!mask || mask[slot] != 0)))
                        v = piece(slot == t.slot ? vn : vc + slot * a.dim, c * L::PIECE);
                    *reinterpret_cast<u32x4 *>(lds + r * L::V_ROW + v_piece<DP>(r, c) * 16) = v;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const int i16 = lane & 15, r = 4 * g + (i16 >> 2);
#pragma unroll
                for (int dt = 0; dt < DP / 16; ++dt) {
                    const int c = 2 * dt + ((i16 >> 1) & 1), byte = 8 * (i16 & 1);
                    const uint2 x = lds_read_transposed(lds + r * L::V_ROW + v_piece<DP>(r, c) * 16 + byte);
                    const uint2 y = lds_read_transposed(lds + (r + 16) * L::V_ROW + v_piece<DP>(r + 16, c) * 16 + byte);
                    V8 code = __builtin_bit_cast(V8, u32x4{x.x, x.y, y.x, y.y});
#pragma unroll
                    for (int i = 0; i < 8; ++i) code[i] = (T)value_code(to_f32(code[i]));
                    const f32x4 count = Mat<T>::mul16(code, one, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int i = 0; i < 4; ++i) held[dt][i] += counted_sum(count[i]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
#pragma unroll
            for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i][r] = held[i][r] == 0.f ? o[i][r] : held[i][r];
        }
    }
    l = quarters_sum(l);
}

// features of accumulator element (tile i, register r) of lane group g
template <class T, int DP> __device__ __forceinline__ int o_feature(int i, int g, int r)
{
    using L = Step<T, DP>;
    return (i / L::VW) * L::SB + L::VW * (4 * g + r) + i % L::VW;
}

// WAVES per task: 4 share a task's slots and join through LDS; 1: a wave has a task of its own, four tasks to a block.
// Narrow tasks of a wave each live on occupancy: 6 waves per SIMD (80 registers) instead of the 5 that the compiler's own choice
// leaves, 26.2 against 29.4 us for one tick of 1600 rows x 8 heads x 51 slots; 8 would spill (45 us).
template <class T, int DP, int WAVES>
__global__ __launch_bounds__(256, WAVES == 1 && DP <= 16 ? 6 : 1) void attn_window_step_kernel(StepArgs a, int head_tiles, int splits, float *part_o, float *part_ml)
{
    using L = Step<T, DP>;
    __shared__ __attribute__((aligned(16))) char lds[4 * L::WAVE_BYTES];
    __shared__ float ml[4][16][2];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned task = WAVES == 4 ? blockIdx.x : blockIdx.x * 4 + wave;      // below 2^31 + 3
    const int split = (int)(task % (unsigned)splits);
    const unsigned r0 = task / (unsigned)splits, r1 = r0 / (unsigned)head_tiles;
    const int ht = (int)(r0 % (unsigned)head_tiles);
    Part t;
    t.kvh = (int)(r1 % (unsigned)a.hk);
    t.b = r1 / (unsigned)a.hk;
    if (t.b >= a.batch) return;
    t.heads = a.group - 16 * ht < 16 ? a.group - 16 * ht : 16;
    t.head0 = t.kvh * a.group + 16 * ht;
    t.p = a.lengths[t.b];
    if (t.p > kMaxLength) t.p = -1;
    t.n = t.p < 0 ? 0 : (t.p < a.slots ? t.p + 1 : a.slots);
    t.slot = t.p < 0 ? -1 : cache_slot(t.p, a.sinks, a.window);
    // equal parts of what is filled, in whole block strides
    const int64_t stride = L::CHUNK * WAVES, per = ((t.n + splits - 1) / splits + stride - 1) / stride * stride;
    t.c0 = split * per;
    t.c1 = t.c0 + per < t.n ? t.c0 + per : t.n;

    f32x4 o[DP / 16];
    float m, l;
    attend_slots<T, DP>(a, t, WAVES == 4 ? wave : 0, WAVES, lane, lds + wave * L::WAVE_BYTES, o, m, l);

    T *out = reinterpret_cast<T *>(a.out) + t.b * (int64_t)a.hq * a.dim;
    if constexpr (WAVES == 1) {
        const float inv = inverse_sum(l);
        if (n < t.heads) {
#pragma unroll
            for (int sb = 0; sb < L::NSB; ++sb)
#pragma unroll
                for (int part = 0; part < L::VW; ++part) {
                    const int d = sb * L::SB + 4 * L::VW * g + 4 * part;
                    Pack<T, 4> w;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int f = 4 * part + x;
                        w.e[x] = from_f32<T>(o[sb * L::VW + f % L::VW][f / L::VW] * inv);
                    }
                    if (d < a.dim) *reinterpret_cast<Pack<T, 4> *>(out + (t.head0 + n) * (int64_t)a.dim + d) = w;
                }
        }
    } else {
        float *mine = reinterpret_cast<float *>(lds + wave * L::WAVE_BYTES);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) mine[n * L::O_STRIDE + o_feature<T, DP>(i, g, r)] = o[i][r];
        if (g == 0) { ml[wave][n][0] = m; ml[wave][n][1] = l; }
        __syncthreads();
        for (int i = threadIdx.x; i < t.heads * a.dim; i += 256) {
            const int hd = i / a.dim, d = i % a.dim;
            float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][hd][0]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float mw = ml[w][hd][0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
                sum = fmaf(f, ml[w][hd][1], sum);
                const float x = reinterpret_cast<float *>(lds + w * L::WAVE_BYTES)[hd * L::O_STRIDE + d];
                // an infinity is one however small its wave's share
                if (mw != -INFINITY) acc = fabsf(x) < INFINITY ? fmaf(f, x, acc) : acc + x;
            }
            const int64_t row = t.b * a.hq + t.head0 + hd;
            if (splits == 1) {
                out[(t.head0 + hd) * (int64_t)a.dim + d] = from_f32<T>(sum == 0.f ? 0.f : acc / sum);
            } else {
                part_o[(row * splits + split) * a.dim + d] = acc;
                if (d == 0) { part_ml[2 * (row * splits + split)] = top; part_ml[2 * (row * splits + split) + 1] = sum; }
            }
        }
    }
    // one wave stores the new token
    if (split == 0 && ht == 0 && t.p >= 0 && (WAVES == 1 || wave == 0)) {
        const T *kn = reinterpret_cast<const T *>(a.k) + t.b * a.kr.tok + t.kvh * a.kr.head;
        const T *vn = reinterpret_cast<const T *>(a.v) + t.b * a.vr.tok + t.kvh * a.vr.head;
        const int64_t to = ((t.b * a.hk + t.kvh) * a.slots + t.slot) * a.dim;
        for (int d = lane; d < a.dim; d += 64) {
            reinterpret_cast<T *>(a.k_cache)[to + d] = kn[d];
            reinterpret_cast<T *>(a.v_cache)[to + d] = vn[d];
        }
        if (t.kvh == 0 && lane == 0 && a.mask_cache) a.mask_cache[t.b * a.slots + t.slot] = !a.key_mask || a.key_mask[t.b] != 0;
    }
}

// Joins the parts of a row: a block per (cache row, query head), its waves take the parts in turn.  All loads of a wave are
// requested before the first is used: the kernel's time is a few memory latencies, not one per part (32 rows in 33 parts: 4.1 us).
constexpr int kMaxSplits = 64;

template <class T>
__global__ __launch_bounds__(256) void attn_window_step_join_kernel(StepArgs a, int splits, const float *__restrict__ part_o,
                                                                    const float *__restrict__ part_ml)
{
    __shared__ float2 acc[4][64];
    const int lane = threadIdx.x & 63, d = 2 * lane;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x, first = row * splits;
    const bool has = d < a.dim;
    const float2 *po = reinterpret_cast<const float2 *>(part_o + first * a.dim + (has ? d : 0));
    const int64_t stride = a.dim / 2;
    const float2 own = lane < splits ? reinterpret_cast<const float2 *>(part_ml)[first + lane] : make_float2(-INFINITY, 0.f);
    float top = own.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    // weight of part `lane`; a part that saw nothing has no numerators
    const float f = own.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own.x - top);
    const float sum = wave_sum(f * own.y);
    constexpr int AHEAD = 8;
    float x = 0.f, y = 0.f;
    for (int s0 = wave; s0 < splits; s0 += 4 * AHEAD) {
        float2 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + 4 * i;
            v[i] = po[(int64_t)(s < splits ? s : s0) * stride];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + 4 * i;
            const float g = __shfl(f, s < splits ? s : 0), mg = __shfl(own.x, s < splits ? s : 0);
            if (s < splits && mg != -INFINITY) {
                x = fabsf(v[i].x) < INFINITY ? fmaf(g, v[i].x, x) : x + v[i].x;
                y = fabsf(v[i].y) < INFINITY ? fmaf(g, v[i].y, y) : y + v[i].y;
            }
        }
    }
    acc[wave][lane] = make_float2(x, y);
    __syncthreads();
    if (wave == 0 && has) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        x = ((acc[0][lane].x + acc[1][lane].x) + (acc[2][lane].x + acc[3][lane].x)) * inv;
        y = ((acc[0][lane].y + acc[1][lane].y) + (acc[2][lane].y + acc[3][lane].y)) * inv;
        Pack<T, 2> two = {{from_f32<T>(x), from_f32<T>(y)}};
        *reinterpret_cast<Pack<T, 2> *>(reinterpret_cast<T *>(a.out) + row * a.dim + d) = two;
    }
}

struct Plan {
    int waves, head_tiles, splits;
};

// A cache of up to 256 slots is eight chunks at most: a wave of its own is enough, and four of them need not wait for each other
// (1600 x 8 heads of 16 in float32: 100 slots 43 us, 76 with a block per task; 240 slots 81, block 100; 64 x 8 heads of 128 in
// bfloat16: 240 slots 25.4 both ways, 500 slots 44, block 28).  Above, a block per task; with few tasks the slots are split further
// as long as there are no more than two blocks per CU, down to 128 slots (one chunk per wave).  4100 slots of 128 in bfloat16, us
// at one, two and four blocks per CU: 4 x 8 key heads 25.1, 23.5, 28.9; 16 x 8: 58.2, 53.4, 59.3; 64 x 8 have two blocks per CU
// undivided: 168 against 182 in two parts.  The plan depends on sizes only, never on the lengths, which are on the device.
Plan plan_step(int64_t batch, int hk, int group, int64_t slots)
{
    Plan p = {slots <= 256 ? 1 : 4, (group + 15) / 16, 1};
    if (p.waves == 4) {
        const int64_t tasks = batch * hk * p.head_tiles, want = 2 * (int64_t)qcn_num_cus();
        int64_t s = tasks > 0 ? want / tasks : 1;
        if (s > (slots + 127) / 128) s = (slots + 127) / 128;
        if (s > kMaxSplits) s = kMaxSplits;
        p.splits = (int)(s < 1 ? 1 : s);
    }
    return p;
}

template <class T, int DP>
int launch_step_dim(const StepArgs &a, const Plan &p, float *ws, hipStream_t s)
{
    const int64_t tasks = a.batch * a.hk * p.head_tiles * p.splits, blocks = p.waves == 4 ? tasks : (tasks + 3) / 4;
    if (tasks >= ((int64_t)1 << 31) || blocks > kMaxBlocks || (p.splits > 1 && a.batch * a.hq > kMaxBlocks)) return QCN_ERR_UNSUPPORTED;
    const int64_t rows = a.batch * a.hq * p.splits;
    float *part_o = ws, *part_ml = ws ? ws + rows * a.dim : nullptr;
    if (p.waves == 4)
        hipLaunchKernelGGL((attn_window_step_kernel<T, DP, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a, p.head_tiles, p.splits, part_o, part_ml);
    else
        hipLaunchKernelGGL((attn_window_step_kernel<T, DP, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a, p.head_tiles, p.splits, part_o, part_ml);
    QCN_CHECK_LAUNCH();
    if (p.splits > 1) {
        hipLaunchKernelGGL(attn_window_step_join_kernel<T>, dim3((unsigned)(a.batch * a.hq)), dim3(256), 0, s, a, p.splits, part_o, part_ml);
        QCN_CHECK_LAUNCH();
    }
    return QCN_OK;
}

template <class T>
int launch_step(const StepArgs &a, const Plan &p, float *ws, hipStream_t s)
{
    if (a.dim <= 16) return launch_step_dim<T, 16>(a, p, ws, s);
    if (a.dim <= 32) return launch_step_dim<T, 32>(a, p, ws, s);
    if (a.dim <= 64) return launch_step_dim<T, 64>(a, p, ws, s);
    if (a.dim <= 96) return launch_step_dim<T, 96>(a, p, ws, s);
    return launch_step_dim<T, 128>(a, p, ws, s);
}

bool cache_shape_ok(int64_t window, int64_t sinks) { return window >= 1 && sinks >= 0 && window < ((int64_t)1 << 40) && sinks < ((int64_t)1 << 40); }

}  // namespace

extern "C" int qcn_window_cache_append(const qcn_window_cache_append_args *args, void *stream)
{
    if (!args) return QCN_ERR_INVALID_ARGUMENT;
    const qcn_window_cache_append_args &x = *args;
    if (x.n_seq < 0 || x.n_tokens < 0 || x.n_kv_heads < 1 || !cache_shape_ok(x.window, x.sinks) || !dtype_known(x.dtype) ||
        (x.key_mask && !x.mask_cache))
        return QCN_ERR_INVALID_ARGUMENT;
    if (x.dim < 8 || x.dim > kMaxDim || x.dim % 8 || x.n_kv_heads > kMaxHeads) return QCN_ERR_UNSUPPORTED;
    if (x.n_tokens == 0 || x.n_seq == 0) return QCN_OK;
    if (!x.k || !x.v || !x.cu || !x.lengths || !x.k_cache || !x.v_cache) return QCN_ERR_INVALID_ARGUMENT;
    if (!rows_aligned(x.k, x.k_strides[0], x.k_strides[1], x.dtype) || !rows_aligned(x.v, x.v_strides[0], x.v_strides[1], x.dtype) ||
        !rows_aligned(x.k_cache, 0, 0, x.dtype) || !rows_aligned(x.v_cache, 0, 0, x.dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    const int64_t blocks = (x.n_tokens >> kAppendShift) + x.n_seq + 1;
    if (x.n_tokens >= ((int64_t)1 << 40) || x.n_seq >= ((int64_t)1 << 31) || blocks > kMaxBlocks) return QCN_ERR_UNSUPPORTED;
    const AppendArgs a = {x.k, x.v, {x.k_strides[0], x.k_strides[1]}, {x.v_strides[0], x.v_strides[1]}, x.cu, x.lengths, x.key_mask,
                          x.n_seq, x.n_tokens, (int)x.n_kv_heads, (int)x.dim, (int)x.dim * (int)dtype_bytes(x.dtype) / 16, x.window,
                          x.sinks, x.window + x.sinks, x.k_cache, x.v_cache, x.mask_cache};
    hipStream_t s = qcn_stream(stream);
    if (x.dtype == QCN_DTYPE_F32)
        hipLaunchKernelGGL(window_cache_append_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    else   // moved as they are: one form for both 16-bit types
        hipLaunchKernelGGL(window_cache_append_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

extern "C" size_t qcn_attn_window_step_workspace_bytes(int64_t batch, int64_t n_q_heads, int64_t n_kv_heads, int64_t dim, int64_t window,
                                                       int64_t sinks)
{
    if (batch < 1 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || n_q_heads > kMaxHeads || dim < 1 ||
        !cache_shape_ok(window, sinks))
        return 0;
    const Plan p = plan_step(batch, (int)n_kv_heads, (int)(n_q_heads / n_kv_heads), window + sinks);
    return p.splits > 1 ? (size_t)batch * n_q_heads * p.splits * (dim + 2) * sizeof(float) : 0;
}

extern "C" int qcn_attn_window_step(const qcn_attn_window_step_args *args, void *stream)
{
    if (!args) return QCN_ERR_INVALID_ARGUMENT;
    const qcn_attn_window_step_args &x = *args;
    if (x.batch < 0 || x.n_q_heads < 1 || x.n_kv_heads < 1 || x.n_q_heads % x.n_kv_heads || !cache_shape_ok(x.window, x.sinks) ||
        !(x.scale >= 0.) || x.scale > kMaxScale || !dtype_known(x.dtype) || (x.key_mask && !x.mask_cache))
        return QCN_ERR_INVALID_ARGUMENT;
    if (x.dim < 8 || x.dim > kMaxDim || x.dim % 8 || x.n_q_heads > kMaxHeads || x.batch >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    if (x.batch == 0) return QCN_OK;
    if (!x.q || !x.k || !x.v || !x.lengths || !x.k_cache || !x.v_cache || !x.out) return QCN_ERR_INVALID_ARGUMENT;
    if (!rows_aligned(x.q, x.q_strides[0], x.q_strides[1], x.dtype) || !rows_aligned(x.k, x.k_strides[0], x.k_strides[1], x.dtype) ||
        !rows_aligned(x.v, x.v_strides[0], x.v_strides[1], x.dtype) || !rows_aligned(x.k_cache, 0, 0, x.dtype) ||
        !rows_aligned(x.v_cache, 0, 0, x.dtype) || !rows_aligned(x.out, 0, 0, x.dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    const int group = (int)(x.n_q_heads / x.n_kv_heads);
    const Plan plan = plan_step(x.batch, (int)x.n_kv_heads, group, x.window + x.sinks);
    const size_t need = qcn_attn_window_step_workspace_bytes(x.batch, x.n_q_heads, x.n_kv_heads, x.dim, x.window, x.sinks);
    if (need && (x.workspace_bytes < (int64_t)need || !x.workspace || ((uintptr_t)x.workspace & 7))) return QCN_ERR_WORKSPACE_TOO_SMALL;
    const StepArgs a = {x.q, x.k, x.v, {x.q_strides[0], x.q_strides[1]}, {x.k_strides[0], x.k_strides[1]}, {x.v_strides[0], x.v_strides[1]},
                        x.lengths, x.key_mask, x.batch, (int)x.n_q_heads, (int)x.n_kv_heads, group, (int)x.dim, x.window, x.sinks,
                        x.window + x.sinks,
                        // an unseen slot's score is -inf and has to stay so: scale 0 becomes one that no score outgrows
                        fmaxf((float)x.scale * kLog2e, 1e-37f), x.k_cache, x.v_cache, x.mask_cache, x.out};
    float *ws = need ? reinterpret_cast<float *>(x.workspace) : nullptr;
    hipStream_t s = qcn_stream(stream);
    switch (x.dtype) {
    case QCN_DTYPE_F32: return launch_step<float>(a, plan, ws, s);
    case QCN_DTYPE_F16: return launch_step<_Float16>(a, plan, ws, s);
    default: return launch_step<__bf16>(a, plan, ws, s);
    }
}
