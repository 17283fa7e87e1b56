// Attention over ragged token sequences with a sliding window and a few first tokens that stay visible (sinks).
//
// Query i of a sequence with Lq queries and Lk keys stands at position p = i + Lk - Lq (the queries are the last of the keys).
// It sees key j when  0 <= j <= p  and  (j > p - window  or  j < sinks)  and key_mask[j]:
//   o = sum_j softmax_j(scale q . k_j) v_j,   o = 0 for a row that sees nothing.
// Hkv key heads are shared by Hq / Hkv query heads each.
//
// The work is 4 dim operations per visible (query, key) pair and head; q, k, v and o pass memory once.  Short windows (an agent's
// 10 steps of 16 features) are bound by memory and its latency, long ones by the matrix units, so there are two kernels:
//   direct  16 rows per wave, operands straight from memory, no barrier: float32, and 16-bit rows of up to 16 features (up to 32
//           where the window is short)
//   tile    128 rows per block, 64-key tiles through LDS: wider 16-bit rows
// Both keep one running maximum and sum per row, in float32, and go over the keys once; a second time only where a value is not
// finite (one that some rows of a wave see and others do not reaches the others as 0 * inf).  Formed again row by row and key by key, as
// they were before, such rows made a call hundreds of times as long (16384 x 16 heads of 128, window 1024, one infinite value in the
// first token: 101 ms, now 0.59; none: 0.16).
#include "sequence.hip.h"

#include <type_traits>

namespace {

using namespace qcn_seq;

struct Args {
    const void *q, *k, *v;
    Rows qr, kr, vr;
    const int64_t *cu_q, *cu_k;
    const uint8_t *key_mask;
    int64_t n_seq, nq, nk;
    int hq, hk, group, dim;
    int64_t window, sinks;
    float c2;             // scale in base 2
    void *out;            // [nq, hq, dim] contiguous
};

// Rows behind the last sequence (and of sequences that see nothing): zero.
template <class T>
__device__ __forceinline__ void zero_row(const Args &a, int64_t row, int head, int lane, int lanes)
{
    T *o = reinterpret_cast<T *>(a.out) + (row * a.hq + head) * (int64_t)a.dim;
    for (int d = lane; d < a.dim; d += lanes) o[d] = from_f32<T>(0.f);
}

// A tile is 2^SHIFT consecutive ROWS of one sequence and one key head; a row is a (query, query head of the group) pair, heads
// fastest: shared keys are read once for the whole group, and a short chunk of queries still fills the tile.
struct Tile {
    int64_t q_beg, k_beg;   // first token of the sequence
    int64_t rows, row0;     // rows of the sequence; first row of the tile
    int lk, shift;          // keys of the sequence; position of query i = i + shift
    int token0, sub0;       // token of the tile's first row (counted in the sequence) and its query head in the group
    bool behind;            // rows behind the last sequence
    // token and query head of the tile's row r
    __device__ __forceinline__ int token(int r, int group) const { return group == 1 ? token0 + r : token0 + (int)((unsigned)(sub0 + r) / (unsigned)group); }
    __device__ __forceinline__ int sub(int r, int group) const { return group == 1 ? 0 : (int)((unsigned)(sub0 + r) % (unsigned)group); }
};

__device__ __forceinline__ Tile find_tile(const Args &a, int64_t tile, int64_t n_tiles, int shift, int lane)
{
    Tile t;
    const Found f = find_seq(a.cu_q, a.n_seq, a.nq, a.group, shift, tile, n_tiles, lane);
    t.behind = f.b == a.n_seq;
    t.q_beg = f.beg;
    int64_t k_end = f.end;
    t.k_beg = f.beg;
    if (t.behind) t.k_beg = k_end = 0;
    else if (a.cu_k != a.cu_q) seq_range(a.cu_k, f.b, a.nk, t.k_beg, k_end);
    else if (k_end > a.nk) { t.k_beg = t.k_beg < a.nk ? t.k_beg : a.nk; k_end = a.nk; }
    t.rows = (f.end - f.beg) * a.group;
    t.row0 = (tile - ((f.beg * a.group >> shift) + f.b)) << shift;
    t.lk = (int)(k_end - t.k_beg);
    t.shift = t.lk - (int)(f.end - f.beg);
    t.token0 = (int)(a.group == 1 ? t.row0 : t.row0 / a.group);
    t.sub0 = a.group == 1 ? 0 : (int)(t.row0 % a.group);
    return t;
}

// The keys that the positions p0 .. p1 see, as one index range 0 .. total - 1: the sinks in front of the window, then the window.
struct Keys {
    int sinks, start, total;
    __device__ __forceinline__ int key(int j) const { return j < sinks ? j : j - sinks + start; }
};

// What one row sees of that range:  [0, sinks)  and  [lo, hi).
struct Sees {
    int sinks, lo, hi;
    // bits of the 64 indexes from j0 on
    static __device__ __forceinline__ uint64_t below(int n) { return n <= 0 ? 0 : (n >= 64 ? ~0ull : (1ull << n) - 1); }
    __device__ __forceinline__ uint64_t bits(int j0) const { return below(sinks - j0) | (below(hi - j0) & ~below(lo - j0)); }
};

__device__ __forceinline__ int window_start(const Args &a, int p) { return a.window > (int64_t)p ? 0 : (int)(p + 1 - a.window); }

__device__ __forceinline__ Keys key_range(const Args &a, int p0, int p1)
{
    Keys k;
    k.start = p0 < 0 ? 0 : window_start(a, p0);
    k.sinks = a.sinks < k.start ? (int)a.sinks : k.start;
    k.total = p1 < 0 ? 0 : k.sinks + p1 + 1 - k.start;
    return k;
}

// Sinks in front of the window keep their own index, and so do those inside it (then the range starts at the window, sinks
// reaching into it, and index = key): either way the sinks up to p are the first min(sinks, p + 1) indexes.
__device__ __forceinline__ Sees row_sees(const Args &a, const Keys &k, int p)
{
    if (p < 0) return {0, 0, 0};
    return {a.sinks < (int64_t)p + 1 ? (int)a.sinks : p + 1, window_start(a, p) - k.start + k.sinks, p + 1 - k.start + k.sinks};
}

// x where the bit is set, else -inf
__device__ __forceinline__ float seen_or_inf(unsigned bits, int bit, float x)
{
    const int keep = __builtin_amdgcn_sbfe((int)bits, bit, 1);
    return __builtin_bit_cast(float, (__builtin_bit_cast(int, x) & keep) | ((int)0xff800000 & ~keep));
}

// ---------------------------------------------------------------------------------------------------------------------
// 16 rows per wave, keys straight from memory (float32 of every width; narrow rows of the 16-bit types)
// ---------------------------------------------------------------------------------------------------------------------
// A wave is on its own: no barrier.  For short windows (the agents' 10 steps) every key tile is used by two or three row
// tiles at most, so staging would cost more than the cache hits it saves.  A wave keeps its 16 rows and goes through key heads:
// where its sequence lies, what its rows see and the rows' offsets are found once, and (narrow heads) the next head's rows are
// requested while this head's are worked on.
//
// v_mfma_f32_16x16x4_f32: contraction index = lane >> 4.  A lane loads 4 neighbouring features (16 bytes) of its key and feeds
// them to 4 products, so product e of piece c contracts features 16 c + 4 g + e.  V^T tile (sb, e) holds features
// sb SB + VW m + e (m = 0 .. 15): a lane ends with 4 VW neighbouring features of its query.  Wide heads load VW neighbouring
// features of a key for it; of narrow ones that would be loads of 4 or 8 bytes, four times as many instructions as the bytes
// need, so their V comes like K and is turned in a few hundred bytes of LDS of the wave's own.
//
// Weights meet 16-bit V in two products, rounded to its type and with what that left (16 bits of bfloat16, 22 of float16 together):
// these rows wait for memory and for each other's results, not for the matrix units (bfloat16, one product and two: 1600 agents x 59 steps x
// 8 heads of 16 33.9 and 35.4 us, 8 x 2000 steps of 16 62 and 61, float16 800 x 59 of 32 28.8 and 28.5, the second with the pass below for
// values that are not finite; one product of twice the contraction for both was no faster).
//
// Measured: 1600 agents x 59 steps x 8 heads of 16 in float32, window 10 + 1 (193 MB read and written): 47.4 us, 4.1 TB/s, bound by
// the latency of three dependent looks (boundaries, rows, LDS) at three to four waves per SIMD.  Wide float32 rows over long windows:
// 80 Tflop/s of the 154 that a library product reaches (8 x 2000 steps, 8 heads of 64 or 128, window 500: 183 and 371 us); the L1
// cache is what bounds them (73 % of its cycles serve a request, against 57 % of the matrix units'): a load of 16 keys serves 16 rows.
// Whole steps with scalar addresses and no masks did not help (183 -> 202 us at 64 features), 32 rows per wave are left.
template <class T, int DP> struct Direct {
    static constexpr int VW = DP % 64 == 0 ? 4 : (DP % 32 == 0 ? 2 : 1);
    static constexpr int SB = 16 * VW, NSB = DP / SB, NT = DP / 16;
    static constexpr int NU = 2, CHUNK = 16 * NU;          // keys of a step
    static constexpr bool NARROW = DP <= 32;               // V through LDS; registers for the next step's rows
    static constexpr int V_STRIDE = DP + 16 / sizeof(T);   // LDS row: the pad spreads the rows of a read over the banks
    static constexpr int HP = NARROW ? 128 / (DP * (int)sizeof(T)) : 1;                // heads of 128 bytes
    static constexpr int HEAD_ELEMS = 48 * V_STRIDE, WAVE_ELEMS = NARROW ? HP * HEAD_ELEMS : 4;
};

template <class T, int N> struct alignas(sizeof(T) * N) Pack { T e[N]; };

// OFF: byte offset inside one of the tensors; 32 bits where every tensor is below 4 GiB (a load then takes a scalar base).
// Waves per SIMD asked for, against the compiler's own choice, measured before there was a second pass (8 x 2000 float32 steps x 8 heads,
// window 500; us): 16 features four (76.5, own 85), 32 four (119.7, own 123.5), 64 four (183, own 196), 96 its own (390; three: 445), 128
// two (371, own 388); today 70, 119, 182, 369 and 370.  1600 x 59 agent steps of 16 float32: 54.3 -> 51 us; 123 registers, and the form with
// 64-bit offsets keeps eight (36 bytes a lane) in scratch memory.  16-bit rows are faster with the compiler's three (35, four with spills: 43).
template <class T, int DP> constexpr int direct_waves() { return sizeof(T) == 2 || DP == 96 ? 1 : DP <= 64 ? 4 : 2; }

// The 16 rows of a wave over its key heads.  Returns which heads hold values that are not finite (a bit per head, from the 65th on
// shared); AGAIN: the second pass of those.
template <class T, int DP, class OFF, bool AGAIN>
__device__ __forceinline__ uint64_t direct_rows(const Args &a, const Tile &t, int wave, int lane, int h0, int h1, T *turn, uint64_t again)
{
    using L = Direct<T, DP>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NU = L::NU;
    const int n = lane & 15, g = lane >> 4;
    const int64_t row0 = t.row0 + 16 * wave;
    const int last = (int)((t.rows - 1 - row0) < 15 ? (t.rows - 1 - row0) : 15);
    const int r_own = 16 * wave + (n < last ? n : last);   // lanes past the end repeat the last row and do not store
    const int64_t qi = t.token(r_own, a.group);
    const int sub = t.sub(r_own, a.group);                 // query head inside the group
    const int p = (int)qi + t.shift;
    const int p0 = t.token(16 * wave, a.group) + t.shift, p1 = t.token(16 * wave + last, a.group) + t.shift;
    const Keys keys = key_range(a, p0, p1);
    const Sees sees = row_sees(a, keys, p);
    const int chunks = (keys.total + L::CHUNK - 1) / L::CHUNK;

    constexpr int ES = sizeof(T);
    const char *qb = reinterpret_cast<const char *>(a.q) + (t.q_beg * a.qr.tok) * ES;
    const char *kb = reinterpret_cast<const char *>(a.k) + (t.k_beg * a.kr.tok) * ES;
    const char *vb = reinterpret_cast<const char *>(a.v) + (t.k_beg * a.vr.tok) * ES;
    char *ob = reinterpret_cast<char *>(a.out) + (t.q_beg * a.hq) * (int64_t)a.dim * ES;
    const OFF q_off = (OFF)((qi * a.qr.tok + sub * a.qr.head) * ES), o_off = (OFF)((qi * a.hq + sub) * (int64_t)a.dim * ES);
    const uint8_t *mask = a.key_mask ? a.key_mask + t.k_beg : nullptr;

    using P4 = Pack<T, 4>;
    using PV = Pack<T, L::VW>;
    constexpr int NS = L::NARROW ? 1 : 4;                  // V loads of a lane per tile come from its own key, or from four
    struct Place {                                         // of a step's keys
        OFF k[NU], v[NU][NS];
        int sees[NU][4], seen[NU][NS];                     // all bits or none: whether this lane's row sees the score's key; whether
    };                                                     // the key of a V load is inside the range and not masked
    const auto locate = [&](int j0) {
        Place x;
        const uint64_t vis = sees.bits(j0);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int j = j0 + 16 * u + n;
            const bool in = j < keys.total;
            const int key = keys.key(in ? j : keys.total - 1);
            const bool ok = in && (!mask || mask[key] != 0);
            const unsigned seen = (unsigned)__ballot(ok) >> (4 * g);
            const unsigned both = seen & (unsigned)(vis >> (16 * u + 4 * g));
            x.k[u] = (OFF)key * (OFF)(a.kr.tok * ES);
#pragma unroll
            for (int r = 0; r < 4; ++r) x.sees[u][r] = __builtin_amdgcn_sbfe((int)both, r, 1);
            if constexpr (L::NARROW) {
                x.v[u][0] = (OFF)key * (OFF)(a.vr.tok * ES);
                x.seen[u][0] = ok ? -1 : 0;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int jv = j0 + 16 * u + 4 * g + r;
                    x.v[u][r] = (OFF)keys.key(jv < keys.total ? jv : keys.total - 1) * (OFF)(a.vr.tok * ES);
                    x.seen[u][r] = __builtin_amdgcn_sbfe((int)seen, r, 1);
                }
            }
        }
        return x;
    };
    struct Rows16 {                                        // 16-key tiles in registers
        P4 k[NU][DP / 16], v[L::NARROW ? NU : 1][DP / 16];
    };
    const bool padded = a.dim < DP;
    const auto four = [&](const char *base, OFF off, int c) {   // features 16 c + 4 g ..
        const int d = 16 * c + 4 * g;
        P4 x = *reinterpret_cast<const P4 *>(base + (OFF)(off + (OFF)((d < a.dim ? d : 0) * ES)));
        if (padded && d >= a.dim) x = P4{};
        return x;
    };
    const auto value = [&](const Place &x, int kvh, int u, int sb, int r) {
        const int d = sb * L::SB + L::VW * n;
        return *reinterpret_cast<const PV *>(vb + kvh * a.vr.head * ES + (OFF)(x.v[u][r] + (OFF)((d < a.dim ? d : 0) * ES)));
    };
    const auto load = [&](const Place &x, int kvh) {
        Rows16 y;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) y.k[u][c] = four(kb + kvh * a.kr.head * ES, x.k[u], c);
        if constexpr (L::NARROW) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) y.v[u][c] = four(vb + kvh * a.vr.head * ES, x.v[u][0], c);
        }
        return y;
    };
    struct Query { P4 q[DP / 16]; };
    const auto load_q = [&](int kvh) {
        Query y;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) y.q[c] = four(qb + (int64_t)kvh * a.group * a.qr.head * ES, q_off, c);
        return y;
    };
    const float c2 = a.c2;
    // scores, -inf where unseen; returns the largest of the lane's row
    const auto scores = [&](const Place &x, const Rows16 &rows, const Query &q, f32x4 (&s)[NU]) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.k[u][c].e[e], q.q[c].e[e], s[u], 0, 0, 0);
                } else {
                    using V4 = typename Mat<T>::V4;
                    s[u] = Mat<T>::mul16(__builtin_bit_cast(V4, rows.k[u][c]), __builtin_bit_cast(V4, q.q[c]), s[u]);
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float raw = s[u][r];
                const int keep = x.sees[u][r];
                s[u][r] = __builtin_bit_cast(float, (__builtin_bit_cast(int, raw) & keep) | ((int)0xff800000 & ~keep));
                top = fmaxf(top, s[u][r]);
            }
        return quarters_max(top) * c2;
    };
    // p in place of the scores; returns the lane's sum
    const auto softmax = [&](f32x4 (&s)[NU], float m) {
        const float base = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c2, -base));
                sum += s[u][r];
            }
        return sum;
    };
    // bits of x where the key counts, else 0: 0 times what a masked key holds must stay 0
    const auto keep = [&](T x, int bits) {
        if constexpr (F32) return __builtin_bit_cast(float, __builtin_bit_cast(int, x) & bits);
        else return __builtin_bit_cast(T, (uint16_t)(__builtin_bit_cast(uint16_t, x) & bits));
    };
    const auto accumulate = [&](const Place &x, int kvh, const f32x4 (&s)[NU], f32x4 (&o)[L::NT], const T *turned) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int sb = 0; sb < L::NSB; ++sb) {
                PV v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (L::NARROW) {
                        v[r] = *reinterpret_cast<const PV *>(turned + (16 * u + 4 * g + r) * L::V_STRIDE + sb * L::SB + L::VW * n);
                    } else {
                        v[r] = value(x, kvh, u, sb, r);
                        if (mask) {
#pragma unroll
                            for (int e = 0; e < L::VW; ++e) v[r].e[e] = keep(v[r].e[e], x.seen[u][r]);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < L::VW; ++e) {
                    if constexpr (F32) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            o[sb * L::VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r].e[e], s[u][r], o[sb * L::VW + e], 0, 0, 0);
                    } else {
                        typename Mat<T>::V4 va, hi, lo;        // p = hi + lo
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            va[r] = v[r].e[e];
                            hi[r] = from_f32<T>(s[u][r]);
                            lo[r] = from_f32<T>(s[u][r] - to_f32(hi[r]));
                        }
                        o[sb * L::VW + e] = Mat<T>::mul16(va, hi, o[sb * L::VW + e]);
                        o[sb * L::VW + e] = Mat<T>::mul16(va, lo, o[sb * L::VW + e]);
                    }
                }
            }
    };
    // LDS of the wave's own: its accesses are done in order; only the compiler is to keep them apart
    const auto in_order = [&]() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };
    // o / l; whether a row of the wave came out not finite though its weights are numbers: the wave has loaded a value that is not
    // finite, and a row that does not see its key has it as 0 * inf, and a row that does, perhaps, as (a weight too small for a float) * inf
    const auto divide = [&](float l, f32x4 (&o)[L::NT]) {
        l = quarters_sum(l);
        const float inv = inverse_sum(l);
        bool bad = false;
#pragma unroll
        for (int i = 0; i < L::NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                o[i][r] *= inv;
                bad |= !(fabsf(o[i][r]) < INFINITY);
            }
        return __ballot(bad && l == l) != 0;
    };
    // the lane's 4 VW neighbouring features per sb, four at a time, to to(feature)
    const auto write = [&](const f32x4 (&o)[L::NT], auto to) {
#pragma unroll
        for (int sb = 0; sb < L::NSB; ++sb) {
            const int d = sb * L::SB + 4 * L::VW * g;
#pragma unroll
            for (int part = 0; part < L::VW; ++part) {
                if (d + 4 * part >= a.dim) break;
                P4 w;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int f = 4 * part + x;            // feature f of the lane's 4 VW: r = f / VW, e = f % VW
                    w.e[x] = from_f32<T>(o[sb * L::VW + f % L::VW][f / L::VW]);
                }
                *reinterpret_cast<P4 *>(to(d + 4 * part)) = w;
            }
        }
    };
    const auto finish = [&](int kvh, float l, f32x4 (&o)[L::NT]) {
        const bool bad = divide(l, o);
        if (n <= last) {
            char *out = ob + (int64_t)kvh * a.group * a.dim * ES;
            write(o, [&](int d) { return out + (OFF)(o_off + (OFF)(d * ES)); });
        }
        return bad;
    };
    const auto clear = [&](f32x4 (&o)[L::NT]) {
#pragma unroll
        for (int i = 0; i < L::NT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    };

    const auto turn_v = [&](const Place &x, const Rows16 &rows) {   // narrow heads: V rows to LDS, masked ones as zeros
        if constexpr (L::NARROW) {
            T *mine = turn + wave * L::WAVE_ELEMS;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    P4 y = rows.v[u][c];
                    if (mask) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) y.e[e] = keep(y.e[e], x.seen[u][0]);
                    }
                    *reinterpret_cast<P4 *>(mine + (16 * u + n) * L::V_STRIDE + 16 * c + 4 * g) = y;
                }
            in_order();
        }
    };
    if constexpr (AGAIN) {
        // Heads whose values are not all finite: once over the keys for maximum and sum, once more with weights that add up to one.  V is
        // taken in two parts: what is finite of it, and the codes of the rest against what each row sees, so that the rest reaches the
        // rows that see it and no other.  Three to four times a head's first pass.
        __builtin_amdgcn_s_waitcnt(0x0F70);                // vmcnt(0): behind the stores of the first pass
        for (int kvh = h0; kvh < h1; ++kvh) {
            if (!((again >> ((kvh - h0) & 63)) & 1)) continue;
            f32x4 s[NU], o[L::NT];
            const Query q = load_q(kvh);
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int step = 0; step < chunks; ++step) {
                const Place x = locate(step * L::CHUNK);
                const float mn = fmaxf(m, scores(x, load(x, kvh), q, s));
                l = l * (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn)) + softmax(s, mn);
                m = mn;
            }
            l = quarters_sum(l);
            // (float16: weights keep to the scale of the largest, as small ones would lose bits, and no sum of them overflows)
            if (!std::is_same_v<T, _Float16> && l > 0.f && l < INFINITY) m += __builtin_amdgcn_logf(l);
            clear(o);
            float sum = 0.f;
#pragma unroll 1
            for (int step = 0; step < chunks; ++step) {
                const Place x = locate(step * L::CHUNK);
                const Rows16 rows = load(x, kvh);
                scores(x, rows, q, s);
                sum += softmax(s, m);
                turn_v(x, rows);
                const T *turned = turn + wave * L::WAVE_ELEMS;
#pragma unroll
                for (int sb = 0; sb < L::NSB; ++sb) {
                    f32x4 count[L::VW];
#pragma unroll
                    for (int e = 0; e < L::VW; ++e) count[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        PV v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if constexpr (L::NARROW) v[r] = *reinterpret_cast<const PV *>(turned + (16 * u + 4 * g + r) * L::V_STRIDE + sb * L::SB + L::VW * n);
                            else v[r] = value(x, kvh, u, sb, r);
                        }
#pragma unroll
                        for (int e = 0; e < L::VW; ++e) {
                            f32x4 &to = o[sb * L::VW + e];
                            using V4 = T __attribute__((ext_vector_type(4)));
                            V4 va, code, hi, lo, one;
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                // (keys that are masked or behind the range are seen by no row)
                                const float c = value_code(to_f32(v[r].e[e]));
                                va[r] = c == 0.f ? v[r].e[e] : (T)0.f;
                                code[r] = (T)c;
                                hi[r] = from_f32<T>(s[u][r]);
                                lo[r] = from_f32<T>(s[u][r] - to_f32(hi[r]));
                                one[r] = (T)(x.sees[u][r] ? 1.f : 0.f);
                            }
                            if constexpr (F32) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    to = __builtin_amdgcn_mfma_f32_16x16x4f32(va[r], s[u][r], to, 0, 0, 0);
                                    count[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(code[r], one[r], count[e], 0, 0, 0);
                                }
                            } else {
                                to = Mat<T>::mul16(va, hi, to);
                                to = Mat<T>::mul16(va, lo, to);
                                count[e] = Mat<T>::mul16(code, one, count[e]);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < L::VW; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[sb * L::VW + e][r] += counted_sum(count[e][r]);
                }
                if constexpr (L::NARROW) in_order();
            }
            finish(kvh, sum, o);
        }
        return 0;
    }
    const auto note = [&](int kvh, bool bad) { again |= bad ? 1ull << ((kvh - h0) & 63) : 0; };

    if constexpr (L::NARROW) {
        if (chunks == 1) {
            // All keys in one step: found once for all heads, and no running maximum.  A load covers 128 bytes of 8 rows, that is
            // as many heads as that takes: with 64 bytes of 16 rows (the operands' own layout) each request fills half a cache
            // line, and the number of requests in flight is what such a wave is short of.  LDS turns rows into operands; the next
            // heads' rows are requested as soon as these are in LDS.
            constexpr int PPH = DP * ES / 16, HP = L::HP, E16 = 16 / ES;     // 16-byte pieces of a head's row, heads, elements
            const int lr = lane >> 3, hp = (lane & 7) / PPH, d = (lane & 7) % PPH * E16;
            const bool past = padded && d >= a.dim;
            const uint64_t vis = sees.bits(0);
            const int jc = lane < keys.total ? lane : keys.total - 1;
            const unsigned seen = (unsigned)__ballot(lane < keys.total && (!mask || mask[keys.key(jc)] != 0));
            Place x = {};
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) x.sees[u][r] = __builtin_amdgcn_sbfe((int)((seen & (unsigned)vis) >> (16 * u + 4 * g)), r, 1);
            OFF qo[2], oo[2], ko[4], vo[4];
            int counts[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = lr + 8 * i, own = 16 * wave + (r < last ? r : last);
                qo[i] = (OFF)((t.token(own, a.group) * a.qr.tok + t.sub(own, a.group) * a.qr.head + (past ? 0 : d)) * ES);
                oo[i] = (OFF)((((int64_t)t.token(own, a.group) * a.hq + t.sub(own, a.group)) * a.dim + d) * ES);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = lr + 8 * i, key = keys.key(j < keys.total ? j : keys.total - 1);
                ko[i] = (OFF)key * (OFF)(a.kr.tok * ES) + (OFF)((past ? 0 : d) * ES);
                vo[i] = (OFF)key * (OFF)(a.vr.tok * ES) + (OFF)((past ? 0 : d) * ES);
                counts[i] = (seen >> j) & 1 ? -1 : 0;
            }
            u32x4 qx[2], kx[4], vx[4];
            const auto request = [&](int first) {
                const int kvh = first + hp < h1 ? first + hp : h1 - 1;
                const OFF qh = (OFF)((int64_t)kvh * a.group * a.qr.head * ES), kh = (OFF)(kvh * a.kr.head * ES), vh = (OFF)(kvh * a.vr.head * ES);
#pragma unroll
                for (int i = 0; i < 2; ++i) qx[i] = *reinterpret_cast<const u32x4 *>(qb + (OFF)(qo[i] + qh));
#pragma unroll
                for (int i = 0; i < 4; ++i) kx[i] = *reinterpret_cast<const u32x4 *>(kb + (OFF)(ko[i] + kh));
#pragma unroll
                for (int i = 0; i < 4; ++i) vx[i] = *reinterpret_cast<const u32x4 *>(vb + (OFF)(vo[i] + vh));
            };
            T *mine = turn + wave * L::WAVE_ELEMS;             // [head][16 rows of q, 32 of k and then of v][V_STRIDE]
            request(h0);
            for (int first = h0; first < h1; first += HP) {
                T *to = mine + hp * L::HEAD_ELEMS + d;
                const u32x4 none = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4 *>(to + (lr + 8 * i) * L::V_STRIDE) = past ? none : qx[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4 *>(to + (16 + lr + 8 * i) * L::V_STRIDE) = past ? none : kx[i];
                in_order();
                Rows16 rows[HP];
                Query q[HP];
#pragma unroll
                for (int i = 0; i < HP; ++i) {
                    const T *own = mine + i * L::HEAD_ELEMS;
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) {
                        q[i].q[c] = *reinterpret_cast<const P4 *>(own + n * L::V_STRIDE + 16 * c + 4 * g);
#pragma unroll
                        for (int u = 0; u < NU; ++u) rows[i].k[u][c] = *reinterpret_cast<const P4 *>(own + (16 + 16 * u + n) * L::V_STRIDE + 16 * c + 4 * g);
                    }
                }
                in_order();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    u32x4 y = vx[i];
                    if (mask) y &= (uint32_t)counts[i];        // 0 times what a masked key holds must stay 0
                    *reinterpret_cast<u32x4 *>(to + (16 + lr + 8 * i) * L::V_STRIDE) = y;
                }
                in_order();
                if (first + HP < h1) request(first + HP);
#pragma unroll
                for (int i = 0; i < HP; ++i) {
                    const int kvh = first + i;
                    if (kvh >= h1) break;
                    const T *own = mine + i * L::HEAD_ELEMS;
                    f32x4 s[NU], o[L::NT];
                    clear(o);
                    const float m = scores(x, rows[i], q[i], s);
                    const float l = softmax(s, m);
                    accumulate(x, kvh, s, o, own + 16 * L::V_STRIDE);
                    note(kvh, divide(l, o));
                    // rows go out as they came in, through the place of q
                    in_order();
                    write(o, [&](int f) { return mine + i * L::HEAD_ELEMS + n * L::V_STRIDE + f; });
                }
                in_order();
                if (first + hp < h1 && !past) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (lr + 8 * i <= last)
                            *reinterpret_cast<u32x4 *>(ob + (OFF)(oo[i] + (OFF)((first + hp) * a.group * a.dim * ES))) =
                                *reinterpret_cast<const u32x4 *>(to + (lr + 8 * i) * L::V_STRIDE);
                }
                in_order();
            }
            return again;
        }
    }
    for (int kvh = h0; kvh < h1; ++kvh) {
        f32x4 s[NU], o[L::NT];
        clear(o);
        float m = -INFINITY, l = 0.f;
        const Query q = load_q(kvh);
        for (int step = 0; step < chunks; ++step) {
            const Place x = locate(step * L::CHUNK);
            const Rows16 rows = load(x, kvh);
            // the maximum follows only jumps of more than 2^8: until then p stays below 2^8 and nothing is rescaled
            const float scaled = scores(x, rows, q, s);
            if (__ballot(scaled > m + 8.f)) {
                const float mn = scaled > m ? scaled : m;
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < L::NT; ++i) o[i] *= alpha;
                m = mn;
            }
            l += softmax(s, m);
            turn_v(x, rows);
            accumulate(x, kvh, s, o, turn + wave * L::WAVE_ELEMS);
            if constexpr (L::NARROW) in_order();
        }
        note(kvh, finish(kvh, l, o));
    }
    return again;
}

template <class T, int DP, class OFF>
__global__ __launch_bounds__(256, (direct_waves<T, DP>())) void attn_window_direct_kernel(Args a, int64_t n_tiles, int heads_per_wave, int head_groups)
{
    using L = Direct<T, DP>;
    __shared__ __attribute__((aligned(16))) T turn[4 * L::WAVE_ELEMS];
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned item = qcn_xcd_remap(blockIdx.x, gridDim.x);
    const int64_t tile = item / (unsigned)head_groups;
    const int h0 = (int)(item % (unsigned)head_groups) * heads_per_wave, h1 = h0 + heads_per_wave < a.hk ? h0 + heads_per_wave : a.hk;
    const Tile t = find_tile(a, tile, n_tiles, 6, lane);
    const int64_t row0 = t.row0 + 16 * wave;
    if (t.row0 < 0 || row0 >= t.rows) return;
    if (t.behind) {
        const int n = lane & 15, r = 16 * wave + n;
        if (row0 + n < t.rows)
            for (int kvh = h0; kvh < h1; ++kvh) zero_row<T>(a, t.q_beg + t.token(r, a.group), kvh * a.group + t.sub(r, a.group), lane >> 4, 4);
        return;
    }
    const uint64_t again = direct_rows<T, DP, OFF, false>(a, t, wave, lane, h0, h1, turn, 0);
    if (again) {
        asm("" : "+v"(lane));   // what the second pass needs of each lane is found again, not kept in registers through the first
        direct_rows<T, DP, OFF, true>(a, t, wave, lane, h0, h1, turn, again);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// 128 rows per block, keys through LDS (16-bit types)
// ---------------------------------------------------------------------------------------------------------------------
// Four waves of 32 rows share tiles of 64 keys, double-buffered in LDS; the next tile's copies (global -> LDS, no registers) are
// in flight while the matrix units work on this one, one barrier per tile.  v_mfma_f32_32x32x16: A = 32 keys (S^T) or 32 features
// (O^T), B = 32 rows.  With the accumulator's row order, k-step t of key half-tile u contracts keys
// 32 u + 16 t + {4 h .. 4 h + 3, 8 + 4 h ..}  in lane half h: V^T is fetched in that order by two transposing LDS reads, P^T is the
// S^T registers rounded to 16 bits: a relative error of at most half a step of the type per weight (bfloat16 2^-8, float16 2^-11); the sum
// takes the rounded weights, so that they add up to one.  The output is rounded to the same type, and its error against 64 bits is 1.4
// times that of a form that keeps the weights (bfloat16 0.0023 against 0.00165, float16 0.00026 against 0.0002).  That is the price of one
// product here: a second one with the remainders, as the direct form and the step have it, costs a quarter of the launch (one and two, us:
// 16384 x 16 heads of 128, window 1024 177 and 222; the ragged prompts below 91 and 112; the chunks 110 and 144).
//
// LDS rows are swizzled in 16-byte pieces so that 16 neighbouring keys' pieces (K) and the 4 x 64 bytes of a transposing read
// (V) cover all 64 banks; the copies write LDS in order and permute their source addresses.
//
// With few blocks (a short chunk of queries behind a long prefix) the key tiles are split over blocks as well and joined by a
// second kernel.
//
// Bound by the matrix units and the vector instructions around them, which two or three waves per SIMD do not fully overlap (an
// earlier state of the kernel, 177 us for 16384 x 16 heads of 128 and window 1024, timed with parts left out: no products 109, no
// LDS reads 151, no exponentials 167, no copies 175).  Measured on a card at work (its first dozen launches after a pause take a tenth
// longer): that case 156 to 167 us a call on different cards, 800 to 857 Tflop/s of the 1130 that a large library product reaches; 24
// ragged prompts up to 2500 x 12 heads of 64, window 512, float16: 87 us, 450 Tflop/s counting visible pairs only (32 rows see 9 or 10
// tiles where one row's window is 8, and 2800 blocks are 3.7 rounds of the card); chunks of 200 to 333 queries x 32 heads of 128 behind
// 7000 keys each, window 4096, in three parts: 105 us with the join, 680 Tflop/s.  Four waves per SIMD at dim 64 spill (103 against 93
// us); at dim 32 they have to be asked for, as the second pass would take 135 registers of the 115 that do (800 x 59 x 8 heads, window
// 30: 52 us, three waves 58).
template <int LS> __device__ __forceinline__ int k_piece(int row, int piece)
{
    return piece ^ (LS == 128 ? row & 15 : LS == 64 ? (row >> 1) & 7 : (row >> 2) & 3);
}
template <int LS> __device__ __forceinline__ int v_piece(int row, int piece)
{
    return piece ^ (LS == 128 ? (row & 3) << 2 : LS == 64 ? ((row >> 1) & 1) << 2 : 0);
}

constexpr int64_t kMost = ((int64_t)1 << 31) - 256;   // positions, and the end of a tile behind the last, are 32-bit
constexpr int kRowShift = 7, kKeys = 64, kMaxSplits = 8;

// 64 x 16 bytes, lane's own source, to LDS bytes dst .. dst + 1023 (dst the same in the wave).  Written out, and not as the builtin:
// the compiler takes every transposing read for a possible reader of every copy in flight and waits for all of them; the copies
// of a step belong to the NEXT step's tiles, and copies_landed() at that step's barrier is the wait they need.  (m0 is a reserved
// register: the compiler sets it in front of each instruction of its own that reads it and keeps nothing there.)
__device__ __forceinline__ void copy_to_lds(const void *base, uint32_t offset, uint32_t dst)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(dst) : "memory");
}
__device__ __forceinline__ void copy_to_lds(const void *src, uint32_t dst)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(dst) : "memory");
}

__device__ __forceinline__ void copies_landed()
{
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
    __syncthreads();
}

__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

template <class T, int DP>
__global__ __launch_bounds__(256, DP == 32 ? 4 : 2) void attn_window_tile_kernel(Args a, int64_t n_tiles, int splits, float *part_o, float *part_ml)
{
    constexpr int LS = DP == 96 ? 128 : DP;                    // elements of an LDS row
    constexpr int PIECES = LS / 8, PER = LS / 32, NK = DP / 16, ND = DP / 32, TILE = kKeys * LS;
    using V8 = typename Mat<T>::V8;
    __shared__ __attribute__((aligned(16))) T lds[4 * TILE];   // K, V of one buffer, K, V of the other
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    unsigned item = qcn_xcd_remap(blockIdx.x, gridDim.x);
    const int split = (int)(item % (unsigned)splits);
    item /= (unsigned)splits;
    const int64_t tile = item % (unsigned)n_tiles;
    const int kvh = (int)(item / (unsigned)n_tiles);
    const Tile t = find_tile(a, tile, n_tiles, kRowShift, lane);
    if (t.row0 < 0 || t.row0 >= t.rows) return;
    const int64_t left = t.rows - 1 - t.row0;
    const int last = (int)(left < 127 ? left : 127);           // last row of the tile
    const int r_local = wave * 32 + n;
    const bool real = r_local <= last;
    const int r_own = real ? r_local : last;
    const int64_t qi = t.token(r_own, a.group);
    const int head = kvh * a.group + t.sub(r_own, a.group);
    const int64_t out_row = (t.q_beg + qi) * a.hq + head;
    if (t.behind) {
        if (splits > 1) {
            if (real && h == 0) { part_ml[2 * (out_row * splits + split)] = -INFINITY; part_ml[2 * (out_row * splits + split) + 1] = 0.f; }
            return;
        }
        for (int r = wave; r <= last; r += 4)
            zero_row<T>(a, t.q_beg + t.token(r, a.group), kvh * a.group + t.sub(r, a.group), lane, 64);
        return;
    }
    const int p = (int)qi + t.shift;
    const int p0 = t.token0 + t.shift, p1 = t.token(last, a.group) + t.shift;
    const Keys keys = key_range(a, p0, p1);
    const Sees sees = row_sees(a, keys, p);
    // the wave's own rows
    const int wa = wave * 32 < last ? wave * 32 : last, wz = wave * 32 + 31 < last ? wave * 32 + 31 : last;
    const int wp0 = t.token(wa, a.group) + t.shift, wp1 = t.token(wz, a.group) + t.shift;
    const int wlo0 = wp0 < 0 ? 0 : window_start(a, wp0), wlo1 = wp1 < 0 ? 0 : window_start(a, wp1);

    const T *q = reinterpret_cast<const T *>(a.q) + (t.q_beg + qi) * a.qr.tok + head * a.qr.head;
    const T *kb = reinterpret_cast<const T *>(a.k) + t.k_beg * a.kr.tok + kvh * a.kr.head;
    const T *vb = reinterpret_cast<const T *>(a.v) + t.k_beg * a.vr.tok + kvh * a.vr.head;
    const uint8_t *mask = a.key_mask ? a.key_mask + t.k_beg : nullptr;

    V8 qf[NK];
#pragma unroll
    for (int c = 0; c < NK; ++c) {
        const int d = 16 * c + 8 * h;
        u32x4 x = *reinterpret_cast<const u32x4 *>(q + (d < a.dim ? d : 0));
        if (d >= a.dim) x = u32x4{0, 0, 0, 0};
        qf[c] = __builtin_bit_cast(V8, x);
    }
    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, l = 0.f, l2 = 0.f;                    // two chains of the sum
    const float c2 = a.c2;
    const int all_steps = (keys.total + kKeys - 1) / kKeys;
    const int per_split = (all_steps + splits - 1) / splits;
    const int s0 = split * per_split, s1 = s0 + per_split < all_steps ? s0 + per_split : all_steps;

    // tiles alternate between two buffers, counted from the first step
    const auto buffer = [&](int parity, int kv) { return lds + (parity * 2 + kv) * TILE; };
    // Copy i of a wave fills 1024 LDS bytes in order, 16 per lane.  Features past the end of a row (dim < DP) are copied from its
    // start: they meet zeros of q, or are never stored.
    const T *k_window = kb + (int64_t)(keys.start - keys.sinks) * a.kr.tok, *v_window = vb + (int64_t)(keys.start - keys.sinks) * a.vr.tok;
    const int r0 = lane / PIECES, slot = lane % PIECES;
    const auto piece = [&](int i, auto want_v) {                // first feature of the lane's 16 bytes
        const int r = (PER * wave + i) * (64 / PIECES) + r0;
        const int d = 8 * (decltype(want_v)::value ? v_piece<LS>(r, slot) : k_piece<LS>(r, slot));
        return d;
    };
    uint32_t k_off[PER], v_off;                                 // bytes; V pieces do not depend on i
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int d = piece(i, std::false_type{});
        k_off[i] = ((uint32_t)r0 * (uint32_t)a.kr.tok + (d < a.dim ? d : 0)) * (uint32_t)sizeof(T);
    }
    {
        const int d = piece(0, std::true_type{});
        v_off = ((uint32_t)r0 * (uint32_t)a.vr.tok + (d < a.dim ? d : 0)) * (uint32_t)sizeof(T);
    }
    const auto load = [&](int step, int parity, auto want_v) {
        constexpr bool V = decltype(want_v)::value;
        const int j0 = step * kKeys;
        const uint32_t dst = lds_address(buffer(parity, V) + PER * wave * 512);
        const int64_t tok = V ? a.vr.tok : a.kr.tok;
        if (j0 >= keys.sinks && j0 + kKeys <= keys.total) {     // 64 neighbouring keys
            const T *x = (V ? v_window : k_window) + (int64_t)(j0 + PER * wave * (64 / PIECES)) * tok;
#pragma unroll
            for (int i = 0; i < PER; ++i, x += 64 / PIECES * tok)
                if (DP == LS || piece(i, want_v) < DP) copy_to_lds(x, V ? v_off : k_off[i], dst + 1024 * i);
        } else {
            const T *src = V ? vb : kb;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int d = piece(i, want_v), j = j0 + (PER * wave + i) * (64 / PIECES) + r0;
                const int jc = j < keys.total ? j : keys.total - 1;
                if (DP == LS || d < DP) copy_to_lds(src + keys.key(jc) * tok + (d < a.dim ? d : 0), dst + 1024 * i);
            }
        }
    };
    // Tiles that any row of the wave sees: those of the sinks, below es, and those of the window, ea .. eb - 1; tiles whose keys all
    // its rows see: f0 .. f1 - 1.  As numbers once, because the loop's scalar instructions are not free.
    const int to_j = keys.sinks - keys.start;                  // window key + to_j = its index
    int es = 0, ea = 0, eb = 0, f0 = 0, f1 = 0;
    if (wp1 >= 0) {
        const int sinks = a.sinks < (int64_t)wp1 + 1 ? (int)a.sinks : wp1 + 1;
        es = (sinks + kKeys - 1) / kKeys;
        ea = (wlo0 + to_j) / kKeys;
        eb = (wp1 + to_j) / kKeys + 1;
        const int fa = wlo1 + to_j > keys.sinks ? wlo1 + to_j : keys.sinks, fb = wp0 + to_j + 1 < keys.total ? wp0 + to_j + 1 : keys.total;
        f0 = (fa + kKeys - 1) / kKeys;
        f1 = mask || wp0 < 0 ? 0 : fb / kKeys;
    }
    // of 64 keys from j0 on, those inside the range and not masked (the same in every wave)
    const auto seen_keys = [&](int j0) {
        const int j = j0 + lane;
        const bool in = j < keys.total;
        return (uint64_t)__ballot(in && (!mask || mask[keys.key(in ? j : 0)] != 0));
    };
    // O^T += V^T P^T, a k-step (16 keys) at a time; its V operands are read a k-step ahead and the next one's exponentials fill
    // the time of its products.  The order is spelled out for the scheduler, which otherwise puts every LDS read right in front of
    // the product that waits for it.
    const auto run_step = [&](int step, auto parity) {
        constexpr int P = decltype(parity)::value;
        copies_landed();                                       // this step's tiles are in LDS, the other buffers are free
        uint64_t seen = ~0ull;
        if (mask) {
            seen = seen_keys(step * kKeys);
            if (seen != ~0ull) {
                // 0 times what a masked key holds must stay 0
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int x = (PER * wave + i) * 64 + lane;
                    if (!((seen >> (x / PIECES)) & 1)) *reinterpret_cast<u32x4 *>(buffer(P, 1) + 8 * x) = u32x4{0, 0, 0, 0};
                }
                __syncthreads();
            }
        }
        if (step + 1 < s1) {
            load(step + 1, P ^ 1, std::false_type{});
            load(step + 1, P ^ 1, std::true_type{});
        }
        if (!(step < es || (step >= ea && step < eb))) return;
        const T *lk = buffer(P, 0), *lv = buffer(P, 1);
        const int i16 = lane & 15;
        V8 kf[NK], vf[2][ND], pb[4];
        f32x16 s[2];
        const auto read_k = [&](int u, int c) {
            const int kr = 32 * u + n;
            kf[c] = *reinterpret_cast<const V8 *>(&lk[kr * LS + 8 * k_piece<LS>(kr, 2 * c + h)]);
        };
        const auto read_v = [&](int k, int dt) {               // k-step k: 16 keys; 32 features
            const int vr = 16 * k + 4 * h + (i16 >> 2), d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
            const uint2 x = lds_read_transposed(&lv[vr * LS + 8 * v_piece<LS>(vr, d >> 3) + (d & 7)]);
            const uint2 y = lds_read_transposed(&lv[(vr + 8) * LS + 8 * v_piece<LS>(vr + 8, d >> 3) + (d & 7)]);
            vf[k & 1][dt] = __builtin_bit_cast(V8, u32x4{x.x, x.y, y.x, y.y});
        };
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
#pragma unroll
        for (int c = 0; c < NK; ++c) read_k(0, c);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            s[0] = Mat<T>::mul32(kf[c], qf[c], s[0]);
            read_k(1, c);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < NK; ++c) {
            s[1] = Mat<T>::mul32(kf[c], qf[c], s[1]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) read_v(0, dt);
        if (!(step >= f0 && step < f1)) {                      // scores of what a row does not see
            const uint64_t vis = sees.bits(step * kKeys) & seen;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const unsigned w = (unsigned)(vis >> (32 * u)) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = seen_or_inf(w, (r & 3) + 8 * (r >> 2), s[u][r]);
            }
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 16; ++r) top[r & 3] = fmaxf(fmaxf(top[r & 3], s[0][r]), s[1][r]);
        top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        // the running maximum follows only jumps of more than 2^8: until then p stays below 2^8 and nothing is rescaled
        const float scaled = halves_max(top[0]) * c2;
        if (__ballot(scaled > m + 8.f)) {
            const float mn = scaled > m ? scaled : m;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
            l2 *= alpha;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.f : m;
        const auto exponentials = [&](int k, int first, int end) {
#pragma unroll
            for (int i = first; i < end; ++i)
                pb[k][i] = from_f32<T>(__builtin_amdgcn_exp2f(fmaf(s[k >> 1][8 * (k & 1) + i], c2, -base)));
        };
        exponentials(0, 0, 8);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                __builtin_amdgcn_sched_barrier(0);
                o[dt] = Mat<T>::mul32(vf[k & 1][dt], pb[k], o[dt]);
                if (k < 3) {
                    read_v(k + 1, dt);
                    exponentials(k + 1, dt * 8 / ND, (dt + 1) * 8 / ND);
                }
                // the sum, of the rounded p that O sums too
#pragma unroll
                for (int i = dt * 4 / ND; i < (dt + 1) * 4 / ND; ++i) {
                    if (k & 1) l2 = Mat<T>::add_pair(pb[k], i, l2);
                    else l = Mat<T>::add_pair(pb[k], i, l);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    __shared__ int any_redo;                                   // set at the end, many barriers later (a wave without steps sets nothing)
    if (tid == 0) any_redo = 0;
    if (s0 < s1) {
        load(s0, 0, std::false_type{});
        load(s0, 0, std::true_type{});
        for (int step = s0; step < s1; step += 2) {
            run_step(step, std::integral_constant<int, 0>{});
            if (step + 1 < s1) run_step(step + 1, std::integral_constant<int, 1>{});
        }
    }
    l = halves_sum(l + l2);
    T *out = reinterpret_cast<T *>(a.out) + out_row * a.dim;
    const auto emit = [&]() {
        if (splits > 1) {
            // joined by attn_window_join_kernel: this part's maximum, sum and numerators
            const int64_t at = out_row * splits + split;
            if (real && h == 0) { part_ml[2 * at] = m; part_ml[2 * at + 1] = l; }
            if (real && m != -INFINITY) {
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int d = 32 * i + 8 * x + 4 * h;
                        if (d < a.dim) *reinterpret_cast<f32x4 *>(part_o + at * a.dim + d) = f32x4{o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]};
                    }
            }
            return;
        }
        const float inv = inverse_sum(l);
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) {                      // 16 features: halves hold {0-3, 8-11} and {4-7, 12-15}
                unsigned w[2][2];
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int r = 8 * x + 4 * y + 2 * z;
                        Pack<T, 2> two = {{from_f32<T>(o[i][r] * inv), from_f32<T>(o[i][r + 1] * inv)}};
                        w[y][z] = __builtin_bit_cast(unsigned, two);
                    }
                const auto w0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                const auto w1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                const int d = 32 * i + 16 * x + 8 * h;         // after the exchange a lane holds 8 neighbouring features
                if (real && d < a.dim) *reinterpret_cast<u32x4 *>(out + d) = u32x4{w0[0], w1[0], w0[1], w1[1]};
            }
    };
    // A value that is not finite, of a key that some rows of the wave see and others do not, reaches the others as 0 * inf.  A row whose
    // weights are not numbers either (l) is NaN by itself; where a row ends before DP its last scores are products with the copied
    // start of a key, and only the second pass says.
    f32x16 any = o[0];                                         // not finite if an element is not (an overflow costs a second pass)
#pragma unroll
    for (int i = 1; i < ND; ++i) any += o[i];
    f32x4 four = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) four[r & 3] += any[r];
    const float sum = (four[0] + four[1]) + (four[2] + four[3]);
    const bool redo = __ballot(!(fabsf(sum) < INFINITY) && (l == l || a.dim < DP)) != 0;
    if (redo) any_redo = 1;
    else emit();
    __syncthreads();
    if (!any_redo) return;

    // The second pass over the keys, for such waves: the maximum is known, and so is the scale that makes the weights add up to one.  V is
    // taken in two parts: what is finite of it, and the codes of the rest against what each row sees.  A simple loop: the block's
    // time with it is three to five times that of the first pass alone.
    if (!std::is_same_v<T, _Float16> && l > 0.f && l < INFINITY) m += __builtin_amdgcn_logf(l);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
    for (int step = s0; step < s1; ++step) {
        __syncthreads();                                       // the last tiles have been read
        load(step, 0, std::false_type{});
        load(step, 0, std::true_type{});
        const uint64_t seen = seen_keys(step * kKeys);
        copies_landed();
        T *lk = buffer(0, 0), *lv = buffer(0, 1), *lc = buffer(1, 1);
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
            const int x = (PER * wave + i) * 64 + lane, row = x / PIECES;
            V8 v = *reinterpret_cast<const V8 *>(lv + 8 * x), code;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = (seen >> row) & 1 ? value_code(to_f32(v[e])) : 0.f;
                v[e] = (seen >> row) & 1 && c == 0.f ? v[e] : (T)0.f;
                code[e] = (T)c;
            }
            *reinterpret_cast<V8 *>(lv + 8 * x) = v;
            *reinterpret_cast<V8 *>(lc + 8 * x) = code;
            if (8 * k_piece<LS>(row, x % PIECES) >= a.dim) *reinterpret_cast<u32x4 *>(lk + 8 * x) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
        if (!redo || !(step < es || (step >= ea && step < eb))) continue;
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
            for (int c = 0; c < NK; ++c) {
                const int kr = 32 * u + n;
                s[u] = Mat<T>::mul32(*reinterpret_cast<const V8 *>(&lk[kr * LS + 8 * k_piece<LS>(kr, 2 * c + h)]), qf[c], s[u]);
            }
        }
        const uint64_t vis = sees.bits(step * kKeys) & seen;
        V8 weight[4], one[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned w = (unsigned)(vis >> (32 * (k >> 1))) >> (4 * h);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 8 * (k & 1) + i, bit = (r & 3) + 8 * (r >> 2);
                weight[k][i] = from_f32<T>(__builtin_amdgcn_exp2f(fmaf(seen_or_inf(w, bit, s[k >> 1][r]), c2, -base)));
                one[k][i] = (T)(float)((w >> bit) & 1);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) l = Mat<T>::add_pair(weight[k], i, l);
        }
        const int i16 = lane & 15;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
            f32x16 count;
#pragma unroll
            for (int r = 0; r < 16; ++r) count[r] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int vr = 16 * k + 4 * h + (i16 >> 2), d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
                const int at = vr * LS + 8 * v_piece<LS>(vr, d >> 3) + (d & 7), at8 = (vr + 8) * LS + 8 * v_piece<LS>(vr + 8, d >> 3) + (d & 7);
                const uint2 x = lds_read_transposed(lv + at), y = lds_read_transposed(lv + at8);
                const uint2 cx = lds_read_transposed(lc + at), cy = lds_read_transposed(lc + at8);
                o[dt] = Mat<T>::mul32(__builtin_bit_cast(V8, u32x4{x.x, x.y, y.x, y.y}), weight[k], o[dt]);
                count = Mat<T>::mul32(__builtin_bit_cast(V8, u32x4{cx.x, cx.y, cy.x, cy.y}), one[k], count);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] += counted_sum(count[r]);
        }
    }
    l = halves_sum(l);
    if (redo) emit();
}

// Joins the parts of a row, all requested before the first is used: half a wave per (token, query head) and 16 bytes of a part per
// lane where there are up to four parts, a wave and 8 bytes where there are up to eight.  Bound by memory and its latency: 34 144 rows
// of 128 in three parts, 61 MB.  (With a wave each they took 4 us more of 124 for the whole call; 2048 rows in eight parts take 2 us
// more of 23 with half a wave each.)
template <int PARTS> constexpr int join_features() { return PARTS <= 4 ? 4 : 2; }

template <class T, int PARTS>
__global__ __launch_bounds__(256) void attn_window_join_kernel(Args a, int splits, const float *__restrict__ part_o,
                                                               const float *__restrict__ part_ml)
{
    constexpr int VE = join_features<PARTS>(), LANES = kMaxDim / VE, ROWS = 64 / LANES;   // of a lane, of a row, of a wave
    using Vec = __attribute__((ext_vector_type(VE))) float;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t rows = a.nq * a.hq, row0 = ((int64_t)blockIdx.x * 4 + wave) * ROWS;
    if (row0 >= rows) return;
    const bool real = row0 + lane / LANES < rows;
    const int64_t row = real ? row0 + lane / LANES : row0;
    const int d = VE * (lane % LANES);
    const bool has = d < a.dim;
    float2 ml[PARTS];
    Vec ov[PARTS];
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        const int64_t at = row * splits + (s < splits ? s : 0);
        ml[s] = reinterpret_cast<const float2 *>(part_ml)[at];
        if (s >= splits) ml[s] = make_float2(-INFINITY, 0.f);
        ov[s] = *reinterpret_cast<const Vec *>(part_o + at * a.dim + (has ? d : 0));
        top = fmaxf(top, ml[s].x);
    }
    // a part that saw nothing has no numerators; its sum is 0, or NaN where every score was
    float f[PARTS], sum = 0.f;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        f[s] = ml[s].x != -INFINITY ? __builtin_amdgcn_exp2f(ml[s].x - top) : 0.f;
        sum = fmaf(f[s], ml[s].y, sum);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    Vec x = {};
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        const bool saw = ml[s].x != -INFINITY;
        const float w = f[s] * inv;                            // (weights first: numerators may be as large as a float is)
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float v = ov[s][e];
            // an infinity that the row sees is one however small its part's share
            x[e] = saw ? (fabsf(v) < INFINITY ? fmaf(w, v, x[e]) : x[e] + v) : x[e];
        }
    }
    if (sum != sum) x = sum;                                   // a score that is no number, in a part that has no numerators
    if (has && real) {
        Pack<T, VE> y;
#pragma unroll
        for (int e = 0; e < VE; ++e) y.e[e] = from_f32<T>(x[e]);
        *reinterpret_cast<Pack<T, VE> *>(reinterpret_cast<T *>(a.out) + row * a.dim + d) = y;
    }
}

template <class T, int DP>
int launch_direct(const Args &a, hipStream_t s)
{
    const int64_t tiles = (a.nq * a.group >> 6) + a.n_seq + 1;
    // as many key heads per wave as leave eight blocks per CU: the setup is shared, and the last round of blocks still is a small
    // part of the launch (four: 8-10 % slower where a head has work of its own, 16 the same; 1600 x 59 agent steps: 52.3 us with
    // four, 51.6 with eight, 56 with 16, 97 with a head per wave)
    int hpw = a.hk;
    while (hpw > 1 && tiles * ((a.hk + hpw - 1) / hpw) < 8 * (int64_t)qcn_num_cus()) hpw = (hpw + 1) / 2;
    const int groups = (a.hk + hpw - 1) / hpw;
    const int64_t blocks = tiles * groups;
    if (blocks > kMaxBlocks) return QCN_ERR_UNSUPPORTED;
    const int64_t most = (int64_t)1 << 32, es = sizeof(T);
    const auto bytes = [&](int64_t tokens, int64_t tok, int64_t head, int64_t heads) { return (tokens * tok + heads * head + a.dim) * es; };
    const bool small = bytes(a.nq, a.qr.tok, a.qr.head, a.hq) < most && bytes(a.nk, a.kr.tok, a.kr.head, a.hk) < most &&
                       bytes(a.nk, a.vr.tok, a.vr.head, a.hk) < most && a.nq * a.hq * a.dim * es < most;
    if (small)
        hipLaunchKernelGGL((attn_window_direct_kernel<T, DP, uint32_t>), dim3((unsigned)blocks), dim3(256), 0, s, a, tiles, hpw, groups);
    else
        hipLaunchKernelGGL((attn_window_direct_kernel<T, DP, uint64_t>), dim3((unsigned)blocks), dim3(256), 0, s, a, tiles, hpw, groups);
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

// Parts of the keys: as many as bring the launch to three blocks of the 128-row kernel per CU (two or three fit at once).  Measured at
// two, three, four and six per CU, us: 1067 queries x 8 key heads of 128 behind 7000 keys each, window 4096 (304 blocks undivided) 140,
// 128, 133, 140; 500 x 8 behind 8000: three 65, four 70; 64 x 8 behind 8000: three 23.4, four 22.9.  A part keeps at least 8 key tiles:
// below that its setup and its share of the join cost more than the emptier card.  Sizes only: lengths are on the device.
int plan_splits(const Args &a)
{
    if (a.dim <= 16) return 1;
    const int64_t blocks = ((a.nq * a.group >> kRowShift) + a.n_seq + 1) * a.hk, want = 3 * (int64_t)qcn_num_cus();
    int64_t reach = a.window + a.sinks + 128 / a.group;
    if (reach > a.nk) reach = a.nk;
    int64_t s = (want + blocks - 1) / blocks;
    if (s > reach / (8 * kKeys)) s = reach / (8 * kKeys);
    if (s > kMaxSplits) s = kMaxSplits;
    return s < 1 ? 1 : (int)s;
}

template <class T, int DP>
int launch_tile(const Args &a, void *workspace, int64_t workspace_bytes, hipStream_t s)
{
    const int splits = plan_splits(a);
    const int64_t rows = a.nq * a.hq * splits;
    if (splits > 1 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < rows * (a.dim + 2) * 4)) return QCN_ERR_WORKSPACE_TOO_SMALL;
    const int64_t tiles = (a.nq * a.group >> kRowShift) + a.n_seq + 1, blocks = tiles * a.hk * splits;
    if (blocks > kMaxBlocks) return QCN_ERR_UNSUPPORTED;
    float *part_o = reinterpret_cast<float *>(workspace), *part_ml = splits > 1 ? part_o + rows * a.dim : nullptr;
    hipLaunchKernelGGL((attn_window_tile_kernel<T, DP>), dim3((unsigned)blocks), dim3(256), 0, s, a, tiles, splits, part_o, part_ml);
    QCN_CHECK_LAUNCH();
    if (splits > 1) {
        const int64_t joined = a.nq * a.hq;
        if (splits <= 4)
            hipLaunchKernelGGL((attn_window_join_kernel<T, 4>), dim3((unsigned)((joined + 7) / 8)), dim3(256), 0, s, a, splits, part_o, part_ml);
        else
            hipLaunchKernelGGL((attn_window_join_kernel<T, kMaxSplits>), dim3((unsigned)((joined + 3) / 4)), dim3(256), 0, s, a, splits, part_o,
                               part_ml);
        QCN_CHECK_LAUNCH();
    }
    return QCN_OK;
}

template <class T>
int launch(const Args &a, void *ws, int64_t ws_bytes, hipStream_t s)
{
    if constexpr (sizeof(T) == 4) {
        if (a.dim <= 16) return launch_direct<T, 16>(a, s);
        if (a.dim <= 32) return launch_direct<T, 32>(a, s);
        if (a.dim <= 64) return launch_direct<T, 64>(a, s);
        if (a.dim <= 96) return launch_direct<T, 96>(a, s);
        return launch_direct<T, 128>(a, s);
    } else {
        if (a.dim <= 16) return launch_direct<T, 16>(a, s);
        // 16 rows and all their keys in one step of the direct form: 800 x 59 steps x 8 heads of 32, window 10 + 1, 29 us against the
        // tile kernel's 50; window 30: 53 against 48.  Of 64 features and more the tile kernel is faster there too (37 against 42 us).
        if (a.dim <= 32 && a.window + a.sinks <= 17) return launch_direct<T, 32>(a, s);
        if (a.dim <= 32) return launch_tile<T, 32>(a, ws, ws_bytes, s);
        if (a.dim <= 64) return launch_tile<T, 64>(a, ws, ws_bytes, s);
        if (a.dim <= 96) return launch_tile<T, 96>(a, ws, ws_bytes, s);
        return launch_tile<T, 128>(a, ws, ws_bytes, s);
    }
}

}  // namespace

extern "C" int64_t qcn_attn_window_workspace_bytes(const qcn_attn_window_args *args)
{
    if (!args || args->dtype == QCN_DTYPE_F32 || args->n_q_tokens < 1 || args->n_kv_heads < 1 || args->n_q_heads < args->n_kv_heads) return 0;
    Args a = {};
    a.nq = args->n_q_tokens; a.nk = args->n_k_tokens; a.n_seq = args->n_seq; a.hk = (int)args->n_kv_heads;
    a.group = (int)(args->n_q_heads / args->n_kv_heads); a.dim = (int)args->dim;
    a.window = args->window < kMost ? args->window : kMost;
    a.sinks = args->sinks < kMost ? args->sinks : kMost;
    const int splits = plan_splits(a);
    return splits > 1 ? a.nq * args->n_q_heads * splits * (a.dim + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int qcn_attn_window(const qcn_attn_window_args *args, void *stream)
{
    if (!args) return QCN_ERR_INVALID_ARGUMENT;
    const qcn_attn_window_args &x = *args;
    if (x.n_seq < 0 || x.n_q_tokens < 0 || x.n_k_tokens < 0 || x.n_q_heads < 1 || x.n_kv_heads < 1 || x.n_q_heads % x.n_kv_heads ||
        x.window < 1 || x.sinks < 0 || !(x.scale >= 0.) || x.scale > kMaxScale || !dtype_known(x.dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    const int64_t most = kMost;
    if (x.dim < 8 || x.dim > kMaxDim || x.dim % 8 || x.n_q_heads > kMaxHeads || x.n_q_tokens > most || x.n_k_tokens > most || x.n_seq > most ||
        x.k_strides[0] >= kMaxTokStride || x.v_strides[0] >= kMaxTokStride)
        return QCN_ERR_UNSUPPORTED;
    if (x.n_q_tokens == 0) return QCN_OK;
    if (!x.q || !x.out || !x.cu_q || !x.cu_k || (x.n_k_tokens && (!x.k || !x.v))) return QCN_ERR_INVALID_ARGUMENT;
    if (!rows_aligned(x.q, x.q_strides[0], x.q_strides[1], x.dtype) || !rows_aligned(x.out, 0, 0, x.dtype) ||
        (x.n_k_tokens && (!rows_aligned(x.k, x.k_strides[0], x.k_strides[1], x.dtype) ||
                          !rows_aligned(x.v, x.v_strides[0], x.v_strides[1], x.dtype))))
        return QCN_ERR_INVALID_ARGUMENT;
    // positions are below 2^31: larger windows and sinks mean the same
    const int64_t window = x.window < most ? x.window : most, sinks = x.sinks < most ? x.sinks : most;
    const Args a = {x.q, x.k, x.v, {x.q_strides[0], x.q_strides[1]}, {x.k_strides[0], x.k_strides[1]}, {x.v_strides[0], x.v_strides[1]},
                    x.cu_q, x.cu_k, x.key_mask, x.n_seq, x.n_q_tokens, x.n_k_tokens, (int)x.n_q_heads, (int)x.n_kv_heads,
                    (int)(x.n_q_heads / x.n_kv_heads), (int)x.dim, window, sinks,
                    // an unseen key's score is -inf and has to stay so: scale 0 becomes one that no score outgrows
                    fmaxf((float)x.scale * kLog2e, 1e-37f), x.out};
    hipStream_t s = qcn_stream(stream);
    switch (x.dtype) {
    case QCN_DTYPE_F32: return launch<float>(a, x.workspace, x.workspace_bytes, s);
    case QCN_DTYPE_F16: return launch<_Float16>(a, x.workspace, x.workspace_bytes, s);
    default: return launch<__bf16>(a, x.workspace, x.workspace_bytes, s);
    }
}
