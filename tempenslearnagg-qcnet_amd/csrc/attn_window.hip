// Attention over ragged token sequences with a sliding window and a few first tokens that stay visible (sinks).
//
// Query i of a sequence with Lq queries and Lk keys stands at position p = i + Lk - Lq (the queries are the last of the keys).
// It sees key j when  0 <= j <= p  and  (j > p - window  or  j < sinks)  and key_mask[j]:
//   o = sum_j softmax_j(scale q . k_j) v_j,   o = 0 for a row that sees nothing.
// Hkv key heads are shared by Hq / Hkv query heads each.
#include "sequence.hip.h"

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
    float scale;
    void *out;            // [nq, hq, dim] contiguous
};

// One wave, one row, key by key: the form that is right for every input.
template <class T>
__device__ __forceinline__ void row_by_wave(const Args &a, int64_t k_beg, int64_t p, int64_t row, int head, int lane)
{
    const T *q = reinterpret_cast<const T *>(a.q) + row * a.qr.tok + head * a.qr.head;
    const T *k = reinterpret_cast<const T *>(a.k) + k_beg * a.kr.tok + (head / a.group) * a.kr.head;
    const T *v = reinterpret_cast<const T *>(a.v) + k_beg * a.vr.tok + (head / a.group) * a.vr.head;
    const bool has0 = lane < a.dim, has1 = lane + 64 < a.dim;
    const float q0 = has0 ? to_f32(q[lane]) : 0.f, q1 = has1 ? to_f32(q[lane + 64]) : 0.f;
    WaveRow r;
    const int64_t start = p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    const int64_t ns = a.sinks < start ? a.sinks : start;
    for (int64_t i = 0; i < ns + (p + 1 - start); ++i) {
        const int64_t j = i < ns ? i : start + (i - ns);
        if (a.key_mask && !a.key_mask[k_beg + j]) continue;
        const T *kj = k + j * a.kr.tok, *vj = v + j * a.vr.tok;
        const float dot = (has0 ? q0 * to_f32(kj[lane]) : 0.f) + (has1 ? q1 * to_f32(kj[lane + 64]) : 0.f);
        r.add(wave_sum(dot) * a.scale, has0 ? to_f32(vj[lane]) : 0.f, has1 ? to_f32(vj[lane + 64]) : 0.f);
    }
    T *o = reinterpret_cast<T *>(a.out) + (row * a.hq + head) * (int64_t)a.dim;
    if (has0) o[lane] = from_f32<T>(r.result(0));
    if (has1) o[lane + 64] = from_f32<T>(r.result(1));
}

template <class T>
__global__ __launch_bounds__(256) void attn_window_rows_kernel(Args a)
{
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int64_t tile = item / a.hq;
    const int head = (int)(item % a.hq);
    if (tile > a.nq + a.n_seq) return;
    const int64_t b = find_seq(a.cu_q, a.n_seq, a.nq, 1, 0, tile, lane);
    if (b == a.n_seq) {
        const int64_t row = clamp64(a.cu_q[b], 0, a.nq) + tile - (clamp64(a.cu_q[b], 0, a.nq) + b);
        if (row >= a.nq) return;
        T *o = reinterpret_cast<T *>(a.out) + (row * a.hq + head) * (int64_t)a.dim;
        for (int d = lane; d < a.dim; d += 64) o[d] = from_f32<T>(0.f);
        return;
    }
    int64_t q_beg, q_end, k_beg, k_end;
    seq_range(a.cu_q, b, a.nq, q_beg, q_end);
    seq_range(a.cu_k, b, a.nk, k_beg, k_end);
    const int64_t i = tile - (q_beg + b);
    if (i >= q_end - q_beg) return;
    row_by_wave<T>(a, k_beg, i + (k_end - k_beg) - (q_end - q_beg), q_beg + i, head, lane);
}

template <class T>
int launch(const Args &a, hipStream_t s)
{
    const int64_t items = (a.nq + a.n_seq + 1) * a.hq;
    const int64_t blocks = (items + 3) / 4;
    if (blocks >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(attn_window_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

}  // namespace

extern "C" int qcn_attn_window(const void *q, int64_t q_tok_stride, int64_t q_head_stride, const void *k, int64_t k_tok_stride,
                               int64_t k_head_stride, const void *v, int64_t v_tok_stride, int64_t v_head_stride,
                               const int64_t *cu_q, const int64_t *cu_k, const uint8_t *key_mask, int64_t n_seq, int64_t n_q_tokens,
                               int64_t n_k_tokens, int n_q_heads, int n_kv_heads, int dim, int dtype, int64_t window, int64_t sinks,
                               float scale, void *out, void *stream)
{
    if (n_seq < 0 || n_q_tokens < 0 || n_k_tokens < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || window < 1 ||
        sinks < 0 || !(scale >= 0.f) || scale > 3.0e38f || !dtype_known(dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    if (dim < 8 || dim > kMaxDim || dim % 8) return QCN_ERR_UNSUPPORTED;
    if (n_q_tokens == 0) return QCN_OK;
    if (!q || !out || !cu_q || !cu_k || (n_k_tokens && (!k || !v))) return QCN_ERR_INVALID_ARGUMENT;
    if (n_q_tokens >= ((int64_t)1 << 40) || n_k_tokens >= ((int64_t)1 << 40) || n_seq >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    if (!rows_aligned(q, q_tok_stride, q_head_stride, dtype) || !rows_aligned(out, 0, 0, dtype) ||
        (n_k_tokens && (!rows_aligned(k, k_tok_stride, k_head_stride, dtype) || !rows_aligned(v, v_tok_stride, v_head_stride, dtype))))
        return QCN_ERR_INVALID_ARGUMENT;
    const int64_t reach = (int64_t)1 << 42;   // positions are below 2^40: larger windows and sinks mean the same
    const Args a = {q, k, v, {q_tok_stride, q_head_stride}, {k_tok_stride, k_head_stride}, {v_tok_stride, v_head_stride}, cu_q, cu_k,
                    key_mask, n_seq, n_q_tokens, n_k_tokens, n_q_heads, n_kv_heads, n_q_heads / n_kv_heads, dim,
                    window < reach ? window : reach, sinks < reach ? sinks : reach, scale, out};
    hipStream_t s = qcn_stream(stream);
    switch (dtype) {
    case QCN_DTYPE_F32: return launch<float>(a, s);
    case QCN_DTYPE_F16: return launch<_Float16>(a, s);
    default: return launch<__bf16>(a, s);
    }
}
