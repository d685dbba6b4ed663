// fa_packed.cu -- attention of whole sequences packed behind one another
// (acefa_flash_attn_packed).
//
// One warp per (query row, head): each lane holds D / 32 dims of the query and
// of the running output, the keys are walked one by one with an online softmax
// in log2 units.  Right for every shape and mask; bound by its arithmetic.
#include <cmath>
#include <cstring>

#include "fa_internal.h"
#include "kv8_internal.h"  // find_item
#include "ptx.cuh"

namespace acefa {
namespace {

struct PackedParams {
    const char    *q, *k, *v;
    char          *dst;
    int64_t        q_nb1, q_nb2, k_nb1, k_nb2, v_nb1, v_nb2, d_nb1, d_nb2;  // row, head; dst: head, row
    const int32_t *cu_q, *cu_k;
    int            n_seq, rows_q, rows_kv, Hq, Hkv;
    int            mask, window;
    int            dst_type;
    float          scale_log2;
    int           *dev_err;
    uint64_t       wait_limit_ns;
};

constexpr int kRowsPerCta = 4;

// The rows of sequence s; n_q = n_k = 0 and bad for offsets that are none.
struct Seq {
    int  q0, n_q, k0, n_k;
    bool bad;
};
__device__ __forceinline__ Seq seq_of(const PackedParams &P, int s) {
    const int a = __ldg(P.cu_q + s), b = __ldg(P.cu_q + s + 1), c = __ldg(P.cu_k + s), d = __ldg(P.cu_k + s + 1);
    Seq       r = {a, b - a, c, d - c, false};
    if (a < 0 || b < a || b > P.rows_q || c < 0 || d < c || d > P.rows_kv) {
        r = {0, 0, 0, 0, true};
    }
    return r;
}

// Keys [lo, hi) that query i of the sequence sees.
__device__ __forceinline__ void visible(const PackedParams &P, const Seq &s, int i, int &lo, int &hi) {
    lo = 0, hi = s.n_k;
    if (P.mask == ACEFA_MASK_CAUSAL) {
        hi = min(max(i + s.n_k - s.n_q + 1, 0), s.n_k);
    } else if (P.mask == ACEFA_MASK_WINDOW) {
        lo = min(max(i - P.window, 0), s.n_k);
        hi = (int) min((int64_t) i + P.window + 1, (int64_t) s.n_k);
    }
}

template <int HD, class T>
__global__ void __launch_bounds__(32 * kRowsPerCta) fa_packed_simple(const __grid_constant__ PackedParams P) {
    constexpr int N = HD / 32;
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int s = threadIdx.x; s < P.n_seq; s += blockDim.x) {
            if (seq_of(P, s).bad) {
                atomicCAS(P.dev_err, 0, DEVERR_APPEND_POS);
            }
        }
    }
    int s, item;
    if (!find_item(P.n_seq, blockIdx.x, [&](int i) { return (seq_of(P, i).n_q + kRowsPerCta - 1) / kRowsPerCta; }, s,
                   item)) {
        return;
    }
    const Seq q  = seq_of(P, s);
    const int i  = item * kRowsPerCta + (int) (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int h  = blockIdx.y, hk = h / (P.Hq / P.Hkv);
    if (i >= q.n_q) {
        return;
    }
    int lo, hi;
    visible(P, q, i, lo, hi);
    float    x[N], o[N], m = -INFINITY, l = 0.0f;
    const T *qp = reinterpret_cast<const T *>(P.q + (int64_t) (q.q0 + i) * P.q_nb1 + (int64_t) h * P.q_nb2);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = (float) qp[lane * N + e];
        o[e] = 0.0f;
    }
    for (int j = lo; j < hi; ++j) {
        const T *kp = reinterpret_cast<const T *>(P.k + (int64_t) (q.k0 + j) * P.k_nb1 + (int64_t) hk * P.k_nb2);
        const T *vp = reinterpret_cast<const T *>(P.v + (int64_t) (q.k0 + j) * P.v_nb1 + (int64_t) hk * P.v_nb2);
        float    d  = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            d = fmaf(x[e], (float) kp[lane * N + e], d);
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            d += __shfl_xor_sync(0xffffffffu, d, off);
        }
        d *= P.scale_log2;
        const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.0f : exp2f(m - mn), p = exp2f(d - mn);
        l = l * f + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            o[e] = fmaf((float) vp[lane * N + e], p, o[e] * f);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    char       *out = P.dst + (int64_t) h * P.d_nb1 + (int64_t) (q.q0 + i) * P.d_nb2;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (P.dst_type == ACEFA_TYPE_F32) {
            reinterpret_cast<float *>(out)[lane * N + e] = o[e] * inv;
        } else {
            reinterpret_cast<T *>(out)[lane * N + e] = (T) (o[e] * inv);
        }
    }
}

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace
}  // namespace acefa

using namespace acefa;

extern "C" ACEFA_API int acefa_flash_attn_packed(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                                 const acefa_tensor *dst, const int32_t *cu_q, const int32_t *cu_k,
                                                 int n_seq, int mask, int window, float scale, void *stream) {
    if (!q || !k || !v || !dst || !cu_q) {
        return ACEFA_ERR_NULL;
    }
    if ((q->type != ACEFA_TYPE_F16 && q->type != ACEFA_TYPE_BF16) || k->type != q->type || v->type != q->type ||
        (dst->type != ACEFA_TYPE_F32 && dst->type != q->type)) {
        return ACEFA_ERR_TYPE;
    }
    const int64_t D = q->ne[0], rows_q = q->ne[1], Hq = q->ne[2], rows_kv = k->ne[1], Hkv = k->ne[2];
    constexpr int64_t kMostRows = 1ll << 24;
    if ((D != 64 && D != 128) || Hq < 1 || Hq > 4096 || Hkv < 1 || Hq % Hkv || rows_q < 0 || rows_q > kMostRows ||
        rows_kv < 0 || rows_kv > kMostRows || q->ne[3] != 1 || k->ne[0] != D || k->ne[3] != 1 || v->ne[0] != D ||
        v->ne[1] != rows_kv || v->ne[2] != Hkv || v->ne[3] != 1 || dst->ne[0] != D || dst->ne[1] != Hq ||
        dst->ne[2] != rows_q || dst->ne[3] != 1 || n_seq < 0 || n_seq > 65535 || !std::isfinite(scale) || scale <= 0.0f ||
        (mask != 0 && mask != ACEFA_MASK_CAUSAL && mask != ACEFA_MASK_WINDOW) ||
        (mask == ACEFA_MASK_WINDOW && window < 0)) {
        return ACEFA_ERR_SHAPE;
    }
    if ((rows_q && (!q->data || !dst->data)) || (rows_kv && (!k->data || !v->data))) {
        return ACEFA_ERR_NULL;
    }
    for (const acefa_tensor *t : {q, k, v}) {
        if (t->ne[1] == 0) {
            continue;  // no rows: strides say nothing
        }
        if (t->nb[0] != 2 || !aligned(t->data, 16) || (t->ne[1] > 1 && t->nb[1] % 16) ||
            (t->ne[2] > 1 && t->nb[2] % 16)) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    const size_t es = dst->type == ACEFA_TYPE_F32 ? 4 : 2;
    if ((rows_q && (dst->nb[0] != es || !aligned(dst->data, es))) || (Hq > 1 && dst->nb[1] % es) ||
        (rows_q > 1 && dst->nb[2] % es) || !aligned(cu_q, 4) || !aligned(cu_k, 4)) {
        return ACEFA_ERR_LAYOUT;
    }
    DeviceCtx ctx;
    const int rc = device_ctx(&ctx);
    if (rc != ACEFA_OK) {
        return rc;
    }
    if (rows_q == 0 || n_seq == 0) {
        note_launches(0, 0);
        return ACEFA_OK;
    }
    PackedParams p;
    std::memset(&p, 0, sizeof(p));
    p.q = static_cast<const char *>(q->data), p.k = static_cast<const char *>(k->data);
    p.v = static_cast<const char *>(v->data), p.dst = static_cast<char *>(dst->data);
    p.q_nb1 = (int64_t) q->nb[1], p.q_nb2 = (int64_t) q->nb[2];
    p.k_nb1 = (int64_t) k->nb[1], p.k_nb2 = (int64_t) k->nb[2];
    p.v_nb1 = (int64_t) v->nb[1], p.v_nb2 = (int64_t) v->nb[2];
    p.d_nb1 = (int64_t) dst->nb[1], p.d_nb2 = (int64_t) dst->nb[2];
    p.cu_q = cu_q, p.cu_k = cu_k ? cu_k : cu_q;
    p.n_seq = n_seq, p.rows_q = (int) rows_q, p.rows_kv = (int) rows_kv;
    p.Hq = (int) Hq, p.Hkv = (int) Hkv;
    p.mask = mask, p.window = window;
    p.dst_type      = dst->type;
    p.scale_log2    = scale * kLog2e;
    p.dev_err       = ctx.dev_err;
    p.wait_limit_ns = ctx.wait_limit_ns;
    const dim3 grid((unsigned) (rows_q / kRowsPerCta + n_seq), (unsigned) Hq);
    auto       s = static_cast<cudaStream_t>(stream);
    if (q->type == ACEFA_TYPE_F16) {
        D == 128 ? fa_packed_simple<128, __half><<<grid, 32 * kRowsPerCta, 0, s>>>(p)
                 : fa_packed_simple<64, __half><<<grid, 32 * kRowsPerCta, 0, s>>>(p);
    } else {
        D == 128 ? fa_packed_simple<128, __nv_bfloat16><<<grid, 32 * kRowsPerCta, 0, s>>>(p)
                 : fa_packed_simple<64, __nv_bfloat16><<<grid, 32 * kRowsPerCta, 0, s>>>(p);
    }
    if (cudaGetLastError() != cudaSuccess) {
        return ACEFA_ERR_CUDA;
    }
    note_launches(1, 3);
    return ACEFA_OK;
}
