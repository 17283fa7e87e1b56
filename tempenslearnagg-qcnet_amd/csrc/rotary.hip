// Rotary positions over several axes: feature pair i of every head is turned by t = pos[token, axis(i)] * freqs[i],
//   a' = a cos t - b sin t,   b' = a sin t + b cos t   (inverse: -t, which is also the gradient's rotation).
// Pairs are (x[i], x[i + pairs]) or, interleaved, (x[2 i], x[2 i + 1]); features behind 2 * pairs pass through.
//
// HBM-bound: every element is read and written once.  The angle is formed and reduced to a fraction of a turn in fp64 (a
// position of 10^6 times a frequency near 1 has no correct fraction in fp32: its ulp there is 0.06 rad), once per (token,
// pair) and not per head: a block builds the (cos, sin) table of its tokens in LDS, then streams the rows past it.
// Measured: 94 400 tokens x 16 heads x 16 features in float32 (194 MB read and written) 35.6 us, 5.4 TB/s; 32 000 tokens x 32
// heads x 128 in bfloat16 (525 MB) 95 us, 5.5 TB/s; a copy of a large tensor reaches 4.9 (torch) to 6.1 TB/s (16 bytes per thread, nothing
// else) on this card.  64 tokens of a decoding step: 3.5 us, two memory latencies.
#include "sequence.hip.h"

namespace {

using namespace qcn_seq;

constexpr int kThreads = 256;
constexpr int kTable = 2048;      // (cos, sin) pairs a block can hold: 16 KiB
constexpr int kMaxAxes = 8;

struct Axes {
    int first[kMaxAxes + 1];      // pair range of each axis
};

template <class T, int N> struct alignas(sizeof(T) * N) Vec { T e[N]; };

struct Args {
    const void *in[2];
    void *out[2];
    Rows rows[2];                 // input strides; outputs are contiguous
    int heads[2];
    int64_t n_tokens;
    int dim, pairs, n_axes, tokens_per_block, heads_per_block;
    const void *pos;
    const float *freqs;
    Axes axes;
    int inverse;
};

template <class P>
__device__ __forceinline__ float2 turn(const Args &a, int64_t token, int pair)
{
    int axis = 0;
    while (axis + 1 < a.n_axes && pair >= a.axes.first[axis + 1]) ++axis;
    const double x = (double)reinterpret_cast<const P *>(a.pos)[token * a.n_axes + axis];
    const double rev = x * (double)a.freqs[pair] * 0.15915494309189533577;   // 1 / (2 pi)
    const float frac = (float)(rev - rint(rev));
    float s, c;
    sincospif(2.f * frac, &s, &c);
    return make_float2(c, a.inverse ? -s : s);
}

// VE elements per access.  A unit is VE pairs (two accesses) or, interleaved, VE elements; units behind the pairs copy.
template <class T, class P, int VE, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Args a)
{
    __shared__ float2 table[kTable];
    const int64_t tok0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int ntok = (int)((a.n_tokens - tok0) < a.tokens_per_block ? (a.n_tokens - tok0) : a.tokens_per_block);
    for (int i = threadIdx.x; i < ntok * a.pairs; i += kThreads) table[i] = turn<P>(a, tok0 + i / a.pairs, i % a.pairs);
    __syncthreads();

    const int all_heads = a.heads[0] + a.heads[1];
    const int head0 = (int)blockIdx.y * a.heads_per_block;
    const int nheads = (all_heads - head0) < a.heads_per_block ? (all_heads - head0) : a.heads_per_block;
    const int pair_units = INTERLEAVED ? a.dim / VE : a.pairs / VE;
    const int units = INTERLEAVED ? pair_units : pair_units + (a.dim - 2 * a.pairs) / VE;
    const int total = ntok * nheads * units;
    using V = Vec<T, VE>;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const int u = i % units, th = i / units;
        const int t = th / nheads;
        int h = head0 + th % nheads;
        const int which = h >= a.heads[0];
        h -= which ? a.heads[0] : 0;
        // (selects: an index into the kernel's arguments would be a load per lane, 5 % of the launch)
        const T *src = reinterpret_cast<const T *>(which ? a.in[1] : a.in[0]) + (tok0 + t) * (which ? a.rows[1].tok : a.rows[0].tok) +
                       h * (which ? a.rows[1].head : a.rows[0].head);
        T *dst = reinterpret_cast<T *>(which ? a.out[1] : a.out[0]) + ((tok0 + t) * (which ? a.heads[1] : a.heads[0]) + h) * (int64_t)a.dim;
        const float2 *cs = table + t * a.pairs;
        if (INTERLEAVED) {
            V x = *reinterpret_cast<const V *>(src + u * VE);
#pragma unroll
            for (int e = 0; e + 1 < VE; e += 2) {
                const int pair = (u * VE + e) / 2;
                if (pair < a.pairs) {
                    const float2 r = cs[pair];
                    const float p = to_f32(x.e[e]), q = to_f32(x.e[e + 1]);
                    x.e[e] = from_f32<T>(p * r.x - q * r.y);
                    x.e[e + 1] = from_f32<T>(p * r.y + q * r.x);
                }
            }
            *reinterpret_cast<V *>(dst + u * VE) = x;
        } else if (u < pair_units) {
            V x = *reinterpret_cast<const V *>(src + u * VE), y = *reinterpret_cast<const V *>(src + a.pairs + u * VE);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float2 r = cs[u * VE + e];
                const float p = to_f32(x.e[e]), q = to_f32(y.e[e]);
                x.e[e] = from_f32<T>(p * r.x - q * r.y);
                y.e[e] = from_f32<T>(p * r.y + q * r.x);
            }
            *reinterpret_cast<V *>(dst + u * VE) = x;
            *reinterpret_cast<V *>(dst + a.pairs + u * VE) = y;
        } else {
            const int at = 2 * a.pairs + (u - pair_units) * VE;
            *reinterpret_cast<V *>(dst + at) = *reinterpret_cast<const V *>(src + at);
        }
    }
}

template <class T, class P, int VE>
void launch_ve(const Args &a, bool interleaved, dim3 grid, hipStream_t s)
{
    if (interleaved)
        hipLaunchKernelGGL((rotary_kernel<T, P, VE < 2 ? 2 : VE, true>), grid, dim3(kThreads), 0, s, a);
    else
        hipLaunchKernelGGL((rotary_kernel<T, P, VE, false>), grid, dim3(kThreads), 0, s, a);
}

template <class T, class P>
void launch(const Args &a, int ve, bool interleaved, dim3 grid, hipStream_t s)
{
    constexpr int kMost = 16 / (int)sizeof(T);
    if (ve >= 8 && kMost >= 8) launch_ve<T, P, kMost>(a, interleaved, grid, s);
    else if (ve >= 4) launch_ve<T, P, 4>(a, interleaved, grid, s);
    else if (ve >= 2) launch_ve<T, P, 2>(a, interleaved, grid, s);
    else launch_ve<T, P, 1>(a, interleaved, grid, s);
}

template <class T>
int launch_pos(const Args &a, int pos_type, int ve, bool interleaved, dim3 grid, hipStream_t s)
{
    switch (pos_type) {
    case QCN_POS_F32: launch<T, float>(a, ve, interleaved, grid, s); break;
    case QCN_POS_I32: launch<T, int32_t>(a, ve, interleaved, grid, s); break;
    case QCN_POS_I64: launch<T, int64_t>(a, ve, interleaved, grid, s); break;
    default: return QCN_ERR_INVALID_ARGUMENT;
    }
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

}  // namespace

extern "C" int qcn_rotary_embed(const qcn_rotary_embed_args *args, void *stream)
{
    if (!args) return QCN_ERR_INVALID_ARGUMENT;
    const qcn_rotary_embed_args &x = *args;
    if (x.n_tokens < 0 || x.n_q_heads < 0 || x.n_k_heads < 0 || x.dim < 2 || (x.dim & 1) || x.n_axes < 1 || x.n_axes > kMaxAxes ||
        !dtype_known(x.dtype) || x.pos_type < QCN_POS_F32 || x.pos_type > QCN_POS_I64)
        return QCN_ERR_INVALID_ARGUMENT;
    if (x.dim > 256 || x.n_q_heads > 32767 || x.n_k_heads > 32767 || x.n_tokens >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    Args a = {};
    for (int i = 0; i < x.n_axes; ++i) {
        if (x.sections[i] < 0 || x.sections[i] > x.dim / 2) return QCN_ERR_INVALID_ARGUMENT;
        a.axes.first[i + 1] = a.axes.first[i] + (int)x.sections[i];
    }
    a.pairs = a.axes.first[x.n_axes];
    if (a.pairs < 1 || 2 * a.pairs > x.dim) return QCN_ERR_INVALID_ARGUMENT;
    const int heads = (int)(x.n_q_heads + x.n_k_heads), dim = (int)x.dim;
    if (x.n_tokens == 0 || heads == 0) return QCN_OK;
    if ((x.k == nullptr) != (x.n_k_heads == 0) || !x.pos || !x.freqs || (x.n_q_heads && (!x.q || !x.q_out)) || (x.n_k_heads && !x.k_out))
        return QCN_ERR_INVALID_ARGUMENT;
    a.in[0] = x.q; a.in[1] = x.k; a.out[0] = x.q_out; a.out[1] = x.k_out;
    a.rows[0] = {x.q_strides[0], x.q_strides[1]}; a.rows[1] = {x.k_strides[0], x.k_strides[1]};
    a.heads[0] = (int)x.n_q_heads; a.heads[1] = (int)x.n_k_heads;
    a.n_tokens = x.n_tokens; a.dim = dim; a.n_axes = (int)x.n_axes; a.pos = x.pos; a.freqs = x.freqs; a.inverse = x.inverse != 0;
    const bool interleaved = x.interleaved != 0;

    // widest access that every row, the pairs' second half and the passed-through features are aligned to
    const int es = (int)dtype_bytes(x.dtype);
    int ve = 16 / es;
    const auto fits = [&](int n) {
        if (dim % n || (!interleaved && a.pairs % n)) return false;
        for (int i = 0; i < 2; ++i) {
            if (!a.heads[i]) continue;
            if (a.rows[i].tok < 0 || a.rows[i].head < 0 || a.rows[i].tok % n || a.rows[i].head % n) return false;
            if (((uintptr_t)a.in[i] | (uintptr_t)a.out[i]) & (uintptr_t)(n * es - 1)) return false;
        }
        return true;
    };
    while (ve > 1 && !fits(ve)) ve /= 2;
    if ((interleaved && ve < 2) || !fits(ve)) return QCN_ERR_INVALID_ARGUMENT;   // a pair, or an element, straddles its alignment

    // 16 KiB of rows per block (8 / 16 / 32 / 64 KiB: 37.9 / 36.9 / 39.3 / 41.3 us for 94 400 float32 tokens of 1 KiB, 100 / 98 / 100 /
    // 106 us for 32 000 of 8 KiB) while that leaves blocks for the card; few tokens: the heads are spread over blocks as well
    const int64_t row_bytes = (int64_t)heads * dim * es;
    int tpb = (int)((16 * 1024 + row_bytes - 1) / row_bytes);
    if (tpb > kTable / a.pairs) tpb = kTable / a.pairs;
    const int64_t cus = qcn_num_cus();
    while (tpb > 1 && (x.n_tokens + tpb - 1) / tpb < 4 * cus) tpb /= 2;
    int hpb = heads;
    while (hpb > 4 && (x.n_tokens + tpb - 1) / tpb * ((heads + hpb - 1) / hpb) < 2 * cus) hpb = (hpb + 1) / 2;
    if ((x.n_tokens + tpb - 1) / tpb > kMaxBlocks) return QCN_ERR_UNSUPPORTED;
    a.tokens_per_block = tpb;
    a.heads_per_block = hpb;
    const dim3 grid((unsigned)((x.n_tokens + tpb - 1) / tpb), (unsigned)((heads + hpb - 1) / hpb));
    hipStream_t s = qcn_stream(stream);
    switch (x.dtype) {
    case QCN_DTYPE_F32: return launch_pos<float>(a, (int)x.pos_type, ve, interleaved, grid, s);
    case QCN_DTYPE_F16: return launch_pos<_Float16>(a, (int)x.pos_type, ve, interleaved, grid, s);
    default: return launch_pos<__bf16>(a, (int)x.pos_type, ve, interleaved, grid, s);
    }
}
