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
template <class T>
__global__ __launch_bounds__(256) void window_cache_append_kernel(AppendArgs a)
{
    const int64_t b = find_seq(a.cu, a.n_seq, a.n, 1, kAppendShift, blockIdx.x, threadIdx.x & 63);
    if (b == a.n_seq) return;                               // behind the last sequence: left as they are
    int64_t beg, end;
    seq_range(a.cu, b, a.n, beg, end);
    const int64_t first = ((int64_t)blockIdx.x - ((beg >> kAppendShift) + b)) << kAppendShift;
    const int64_t old = a.lengths[b];
    if (first >= end - beg || old < 0) return;
    const int64_t total = old + (end - beg);
    const int64_t ntok = end - beg - first < (1 << kAppendShift) ? end - beg - first : (1 << kAppendShift);
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
    float scale;
    void *k_cache, *v_cache;
    uint8_t *mask_cache;
    void *out;                    // [batch, hq, dim] contiguous
};

// One wave per row and query head, slot by slot.  The new token is read from the inputs, never from its slot: the slot is being
// written by another wave of this launch.
template <class T>
__global__ __launch_bounds__(256) void attn_window_step_rows_kernel(StepArgs a)
{
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int64_t b = item / a.hq;
    const int head = (int)(item % a.hq);
    if (b >= a.batch) return;
    const int kvh = head / a.group;
    const bool has0 = lane < a.dim, has1 = lane + 64 < a.dim;
    T *o = reinterpret_cast<T *>(a.out) + (b * a.hq + head) * (int64_t)a.dim;
    const int64_t p = a.lengths[b];
    if (p < 0) {                                            // a row that is not in use
        if (has0) o[lane] = from_f32<T>(0.f);
        if (has1) o[lane + 64] = from_f32<T>(0.f);
        return;
    }
    const T *q = reinterpret_cast<const T *>(a.q) + b * a.qr.tok + head * a.qr.head;
    const T *kn = reinterpret_cast<const T *>(a.k) + b * a.kr.tok + kvh * a.kr.head;
    const T *vn = reinterpret_cast<const T *>(a.v) + b * a.vr.tok + kvh * a.vr.head;
    const int64_t base = (b * a.hk + kvh) * a.slots * a.dim;
    T *kc = reinterpret_cast<T *>(a.k_cache) + base, *vc = reinterpret_cast<T *>(a.v_cache) + base;
    const int64_t slot = cache_slot(p, a.sinks, a.window);
    const int64_t n = p + 1 < a.slots ? p + 1 : a.slots;
    const bool new_seen = !a.mask_cache || !a.key_mask || a.key_mask[b] != 0;
    const float q0 = has0 ? to_f32(q[lane]) : 0.f, q1 = has1 ? to_f32(q[lane + 64]) : 0.f;
    WaveRow r;
    for (int64_t c = 0; c < n; ++c) {
        const bool fresh = c == slot;
        if (fresh ? !new_seen : (a.mask_cache && !a.mask_cache[b * a.slots + c])) continue;
        const T *kj = fresh ? kn : kc + c * a.dim, *vj = fresh ? vn : vc + c * a.dim;
        const float dot = (has0 ? q0 * to_f32(kj[lane]) : 0.f) + (has1 ? q1 * to_f32(kj[lane + 64]) : 0.f);
        r.add(wave_sum(dot) * a.scale, has0 ? to_f32(vj[lane]) : 0.f, has1 ? to_f32(vj[lane + 64]) : 0.f);
    }
    if (has0) o[lane] = from_f32<T>(r.result(0));
    if (has1) o[lane + 64] = from_f32<T>(r.result(1));
    if (head % a.group == 0) {
        if (has0) { kc[slot * a.dim + lane] = kn[lane]; vc[slot * a.dim + lane] = vn[lane]; }
        if (has1) { kc[slot * a.dim + lane + 64] = kn[lane + 64]; vc[slot * a.dim + lane + 64] = vn[lane + 64]; }
        if (head == 0 && lane == 0 && a.mask_cache) a.mask_cache[b * a.slots + slot] = new_seen;
    }
}

template <class T>
int launch_step(const StepArgs &a, hipStream_t s)
{
    const int64_t blocks = (a.batch * a.hq + 3) / 4;
    if (blocks >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(attn_window_step_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

bool cache_shape_ok(int64_t window, int64_t sinks) { return window >= 1 && sinks >= 0 && window < ((int64_t)1 << 40) && sinks < ((int64_t)1 << 40); }

}  // namespace

extern "C" int qcn_window_cache_append(const void *k, int64_t k_tok_stride, int64_t k_head_stride, const void *v, int64_t v_tok_stride,
                                       int64_t v_head_stride, const int64_t *cu, const int64_t *lengths, const uint8_t *key_mask,
                                       int64_t n_seq, int64_t n_tokens, int n_kv_heads, int dim, int dtype, int64_t window,
                                       int64_t sinks, void *k_cache, void *v_cache, uint8_t *mask_cache, void *stream)
{
    if (n_seq < 0 || n_tokens < 0 || n_kv_heads < 1 || !cache_shape_ok(window, sinks) || !dtype_known(dtype) || (key_mask && !mask_cache))
        return QCN_ERR_INVALID_ARGUMENT;
    if (dim < 8 || dim > kMaxDim || dim % 8 || n_kv_heads > 65535) return QCN_ERR_UNSUPPORTED;
    if (n_tokens == 0 || n_seq == 0) return QCN_OK;
    if (!k || !v || !cu || !lengths || !k_cache || !v_cache) return QCN_ERR_INVALID_ARGUMENT;
    if (!rows_aligned(k, k_tok_stride, k_head_stride, dtype) || !rows_aligned(v, v_tok_stride, v_head_stride, dtype) ||
        !rows_aligned(k_cache, 0, 0, dtype) || !rows_aligned(v_cache, 0, 0, dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    const int64_t blocks = (n_tokens >> kAppendShift) + n_seq + 1;
    if (n_tokens >= ((int64_t)1 << 40) || blocks >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    const AppendArgs a = {k, v, {k_tok_stride, k_head_stride}, {v_tok_stride, v_head_stride}, cu, lengths, key_mask, n_seq, n_tokens,
                          n_kv_heads, dim, dim * (int)dtype_bytes(dtype) / 16, window, sinks, window + sinks, k_cache, v_cache, mask_cache};
    hipStream_t s = qcn_stream(stream);
    if (dtype == QCN_DTYPE_F32)
        hipLaunchKernelGGL(window_cache_append_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    else   // moved as they are: one form for both 16-bit types
        hipLaunchKernelGGL(window_cache_append_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    QCN_CHECK_LAUNCH();
    return QCN_OK;
}

extern "C" size_t qcn_attn_window_step_workspace_bytes(int64_t batch, int n_q_heads, int n_kv_heads, int dim, int64_t window, int64_t sinks)
{
    (void)batch; (void)n_q_heads; (void)n_kv_heads; (void)dim; (void)window; (void)sinks;
    return 0;
}

extern "C" int qcn_attn_window_step(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k, int64_t k_row_stride,
                                    int64_t k_head_stride, const void *v, int64_t v_row_stride, int64_t v_head_stride,
                                    const int64_t *lengths, const uint8_t *key_mask, int64_t batch, int n_q_heads, int n_kv_heads,
                                    int dim, int dtype, int64_t window, int64_t sinks, float scale, void *k_cache, void *v_cache,
                                    uint8_t *mask_cache, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (batch < 0 || n_q_heads < 1 || n_kv_heads < 1 || n_q_heads % n_kv_heads || !cache_shape_ok(window, sinks) || !(scale >= 0.f) ||
        scale > 3.0e38f || !dtype_known(dtype) || (key_mask && !mask_cache))
        return QCN_ERR_INVALID_ARGUMENT;
    if (dim < 8 || dim > kMaxDim || dim % 8) return QCN_ERR_UNSUPPORTED;
    if (batch == 0) return QCN_OK;
    if (!q || !k || !v || !lengths || !k_cache || !v_cache || !out) return QCN_ERR_INVALID_ARGUMENT;
    if (batch >= ((int64_t)1 << 31)) return QCN_ERR_UNSUPPORTED;
    if (!rows_aligned(q, q_row_stride, q_head_stride, dtype) || !rows_aligned(k, k_row_stride, k_head_stride, dtype) ||
        !rows_aligned(v, v_row_stride, v_head_stride, dtype) || !rows_aligned(k_cache, 0, 0, dtype) ||
        !rows_aligned(v_cache, 0, 0, dtype) || !rows_aligned(out, 0, 0, dtype))
        return QCN_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < qcn_attn_window_step_workspace_bytes(batch, n_q_heads, n_kv_heads, dim, window, sinks) ||
        (workspace_bytes && !workspace))
        return QCN_ERR_WORKSPACE_TOO_SMALL;
    const StepArgs a = {q, k, v, {q_row_stride, q_head_stride}, {k_row_stride, k_head_stride}, {v_row_stride, v_head_stride}, lengths,
                        key_mask, batch, n_q_heads, n_kv_heads, n_q_heads / n_kv_heads, dim, window, sinks, window + sinks, scale,
                        k_cache, v_cache, mask_cache, out};
    hipStream_t s = qcn_stream(stream);
    switch (dtype) {
    case QCN_DTYPE_F32: return launch_step<float>(a, s);
    case QCN_DTYPE_F16: return launch_step<_Float16>(a, s);
    default: return launch_step<__bf16>(a, s);
    }
}
