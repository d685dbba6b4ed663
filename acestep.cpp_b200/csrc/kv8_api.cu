// kv8_api.cu -- the C entries of the 8-bit block-scaled KV cache
// (acefa_kv8_*): argument checks in the manner of fa_api.cu and dispatch.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "kv8_internal.h"

namespace acefa {
namespace {

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

size_t elem_size(int type) {
    return type == ACEFA_TYPE_F32 || type == ACEFA_TYPE_I32 ? 4
           : type == ACEFA_TYPE_F16 || type == ACEFA_TYPE_BF16 ? 2
                                                               : 1;
}
bool is_float(int type) { return type == ACEFA_TYPE_F32 || type == ACEFA_TYPE_F16 || type == ACEFA_TYPE_BF16; }

// Bytes from t's data to behind its last element.
size_t extent(const acefa_tensor &t) {
    size_t b = elem_size(t.type);
    for (int i = 0; i < 4; ++i) {
        b += (size_t) (t.ne[i] - 1) * t.nb[i];
    }
    return b;
}
// No two elements at one address (so that kernels may write it in any order);
// with `twin`, nor one with an element of the same tensor `twin` bytes further on.
bool disjoint(const acefa_tensor &t, size_t twin = 0) {
    size_t nb[5]    = {t.nb[0], t.nb[1], t.nb[2], t.nb[3], twin};
    size_t ne[5]    = {(size_t) t.ne[0], (size_t) t.ne[1], (size_t) t.ne[2], (size_t) t.ne[3], twin ? 2u : 1u};
    int    order[5] = {0, 1, 2, 3, 4};
    size_t next     = elem_size(t.type);
    std::sort(order, order + 5, [&](int a, int b) { return nb[a] < nb[b]; });
    for (int i : order) {
        if (ne[i] == 1) {
            continue;
        }
        if (nb[i] < next) {
            return false;
        }
        next = nb[i] * ne[i];
    }
    return true;
}
// Whether a and b share an address, as far as their extents tell; two of the
// same layout may be interleaved (K and V of one buffer).
bool overlap(const acefa_tensor &a, const acefa_tensor &b) {
    const auto x = reinterpret_cast<uintptr_t>(a.data), y = reinterpret_cast<uintptr_t>(b.data);
    if (!(x < y + extent(b) && y < x + extent(a))) {
        return false;
    }
    bool same = a.type == b.type && x != y;
    for (int i = 0; i < 4; ++i) {
        same = same && a.ne[i] == b.ne[i] && a.nb[i] == b.nb[i];
    }
    return !(same && disjoint(a, x < y ? y - x : x - y));
}

int check_shape(const acefa_tensor &t, int64_t n0, int64_t n1, int64_t n2, int64_t n3) {
    return t.ne[0] == n0 && t.ne[1] == n1 && t.ne[2] == n2 && t.ne[3] == n3 ? ACEFA_OK : ACEFA_ERR_SHAPE;
}
// nb[0] is the element size, the strides of longer dims and the data are multiples of `a`.
int check_layout(const acefa_tensor &t, size_t a) {
    if (t.nb[0] != elem_size(t.type) || !aligned(t.data, a)) {
        return ACEFA_ERR_LAYOUT;
    }
    for (int i = 1; i < 4; ++i) {
        if (t.ne[i] > 1 && t.nb[i] % a) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    return ACEFA_OK;
}

int check_cache(const acefa_kv8_cache *c, bool written, Kv8Dev *d) {
    if (!c || !c->k.data || !c->v.data || !c->k_scale.data || !c->v_scale.data) {
        return ACEFA_ERR_NULL;
    }
    if (c->k.type != ACEFA_TYPE_I8 || c->v.type != ACEFA_TYPE_I8 || c->k_scale.type != ACEFA_TYPE_F32 ||
        c->v_scale.type != ACEFA_TYPE_F32) {
        return ACEFA_ERR_TYPE;
    }
    const int64_t D = c->k.ne[0], n = c->k.ne[1], H = c->k.ne[2], B = c->k.ne[3];
    if ((D != 64 && D != 128) || n < 1 || n > (1ll << 30) || H < 1 || H > 4096 || B < 1 || B > kKv8MaxSets ||
        check_shape(c->v, D, n, H, B) != ACEFA_OK) {
        return ACEFA_ERR_SHAPE;
    }
    const int64_t nb = (n + kKv8Block - 1) / kKv8Block;
    for (const acefa_tensor *t : {&c->k_scale, &c->v_scale}) {
        if (check_shape(*t, nb, H, B, 1) != ACEFA_OK) {
            return ACEFA_ERR_SHAPE;
        }
        if (check_layout(*t, 4) != ACEFA_OK || (written && !disjoint(*t))) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    for (const acefa_tensor *t : {&c->k, &c->v}) {
        if (t->nb[0] != 1 || !aligned(t->data, 16) || (written && !disjoint(*t))) {
            return ACEFA_ERR_LAYOUT;
        }
        for (int i = 1; i < 4; ++i) {  // (no tensor map has a stride of 0)
            if (t->ne[i] > 1 && (t->nb[i] % 16 || t->nb[i] == 0)) {
                return ACEFA_ERR_LAYOUT;
            }
        }
    }
    if (written) {
        const acefa_tensor *all[4] = {&c->k, &c->v, &c->k_scale, &c->v_scale};
        for (int i = 0; i < 4; ++i) {
            for (int j = 0; j < i; ++j) {
                if (overlap(*all[i], *all[j])) {
                    return ACEFA_ERR_LAYOUT;
                }
            }
        }
    }
    auto side = [](const acefa_tensor &q, const acefa_tensor &s) {
        Kv8Side r;
        r.q = static_cast<int8_t *>(q.data), r.scale = static_cast<float *>(s.data);
        r.nb1 = (int64_t) q.nb[1], r.nb2 = (int64_t) q.nb[2], r.nb3 = (int64_t) q.nb[3];
        r.s_nb2 = (int64_t) s.nb[1], r.s_nb3 = (int64_t) s.nb[2];
        return r;
    };
    d->k = side(c->k, c->k_scale), d->v = side(c->v, c->v_scale);
    d->D = (int) D, d->n_max = (int) n, d->Hkv = (int) H, d->B = (int) B;
    return ACEFA_OK;
}

Kv8Rows rows_of(const acefa_tensor &t) {
    return Kv8Rows{static_cast<char *>(t.data), (int64_t) t.nb[1], (int64_t) t.nb[2], (int64_t) t.nb[3], t.type};
}

// F32 / F16 / BF16 of the given shape, dense in its first dim.
int check_rows(const acefa_tensor &t, int64_t n0, int64_t n1, int64_t n2, int64_t n3) {
    if (!is_float(t.type)) {
        return ACEFA_ERR_TYPE;
    }
    if (check_shape(t, n0, n1, n2, n3) != ACEFA_OK) {
        return ACEFA_ERR_SHAPE;
    }
    return n1 == 0 ? ACEFA_OK : check_layout(t, elem_size(t.type));  // no rows: strides say nothing
}

// F32 or I32 [n, Hkv, B] (weights, kept rows)
int check_per_row(const acefa_tensor &t, int type, int64_t n, const Kv8Dev &c, bool written) {
    if (t.type != type) {
        return ACEFA_ERR_TYPE;
    }
    if (check_shape(t, n, c.Hkv, c.B, 1) != ACEFA_OK) {
        return ACEFA_ERR_SHAPE;
    }
    return check_layout(t, 4) != ACEFA_OK || (written && !disjoint(t)) ? ACEFA_ERR_LAYOUT : ACEFA_OK;
}

bool overlaps_cache(const acefa_tensor &t, const acefa_kv8_cache &c) {
    return overlap(t, c.k) || overlap(t, c.v) || overlap(t, c.k_scale) || overlap(t, c.v_scale);
}

struct AttnPlan {
    Kv8AttnParams p;
    size_t        part_bytes, ws_bytes;
};

// Checks of acefa_kv8_attn and the plan: a function of the operands and, for
// the number of CTAs, of the device.
int plan_attn(const acefa_tensor *q, const acefa_kv8_cache *cache, const acefa_tensor *weight, AttnPlan *plan) {
    Kv8AttnParams &p = plan->p;
    std::memset(&p, 0, sizeof(p));
    if (!q || !q->data || (weight && !weight->data)) {
        return ACEFA_ERR_NULL;
    }
    int rc = check_cache(cache, false, &p.c);
    if (rc != ACEFA_OK) {
        return rc;
    }
    const int64_t n_q = q->ne[1], Hq = q->ne[2];
    if (n_q < 1 || n_q > ACEFA_KV8_MAX_ROWS || Hq < 1 || Hq > 4096 || Hq % p.c.Hkv) {
        return ACEFA_ERR_SHAPE;
    }
    if ((rc = check_rows(*q, p.c.D, n_q, Hq, p.c.B)) != ACEFA_OK) {
        return rc;
    }
    if (n_q * (Hq / p.c.Hkv) > ACEFA_KV8_MAX_ROWS) {
        return ACEFA_ERR_SHAPE;
    }
    if (weight) {
        if ((rc = check_per_row(*weight, ACEFA_TYPE_F32, p.c.n_max, p.c, true)) != ACEFA_OK) {
            return rc;
        }
        p.weight = static_cast<char *>(weight->data);
        p.w_nb2 = (int64_t) weight->nb[1], p.w_nb3 = (int64_t) weight->nb[2];
    }
    p.q    = rows_of(*q);
    p.n_q  = (int) n_q;
    p.G    = (int) (Hq / p.c.Hkv);
    p.rows = p.n_q * p.G;
    const int R = kv8_unit_rows(p.rows, q->type);
    p.n_rb      = (p.rows + R - 1) / R;
    const int64_t units = (int64_t) p.c.B * p.c.Hkv * p.n_rb;
    const int64_t tiles = units * ((p.c.n_max + kKv8Block - 1) / kKv8Block);  // places of the kernel: + 2 per unit
    const int64_t weigh = weight ? (int64_t) p.c.B * p.c.Hkv * (p.c.n_max / 256 + 1) : 0;
    if (tiles + 2 * units >= (1ll << 31) || units * R + weigh >= (1ll << 31)) {
        return ACEFA_ERR_SHAPE;
    }
    DeviceCtx ctx;
    if ((rc = device_ctx(&ctx)) != ACEFA_OK) {
        return rc;
    }
    p.n_cta           = (int) std::min<int64_t>(tiles, (int64_t) ctx.sm_count * kv8_attn_ctas_per_sm());
    p.cluster         = kv8_attn_cluster(p, units, ctx.sm_count);
    p.dev_err         = ctx.dev_err;
    p.wait_limit_ns   = ctx.wait_limit_ns;
    p.score_stride    = std::min(R, (p.rows + 1) & ~1);
    plan->part_bytes  = ((size_t) (p.n_cta + units) * kv8_slot_floats(p.c.D, R) * sizeof(float) + 255) / 256 * 256;
    plan->ws_bytes    = plan->part_bytes +
                     (weight ? (size_t) units * (size_t) p.c.n_max * (size_t) p.score_stride * sizeof(float) : 0);
    return ACEFA_OK;
}

}  // namespace
}  // namespace acefa

using namespace acefa;

extern "C" {

ACEFA_API int acefa_kv8_store(const acefa_kv8_cache *cache, const acefa_tensor *k_new, const acefa_tensor *v_new,
                              const int32_t *cu_rows, const int32_t *pos, void *stream) {
    Kv8StoreParams p;
    std::memset(&p, 0, sizeof(p));
    if (!k_new || !v_new || !pos) {
        return ACEFA_ERR_NULL;
    }
    int rc = check_cache(cache, true, &p.c);
    if (rc != ACEFA_OK) {
        return rc;
    }
    const int64_t rows = k_new->ne[1];
    if (rows != 0 && (!k_new->data || !v_new->data)) {
        return ACEFA_ERR_NULL;
    }
    if (v_new->type != k_new->type) {
        return ACEFA_ERR_TYPE;
    }
    if (rows < 0 || rows > (1ll << 30) || (!cu_rows && rows % p.c.B)) {
        return ACEFA_ERR_SHAPE;
    }
    for (const acefa_tensor *t : {k_new, v_new}) {
        if ((rc = check_rows(*t, p.c.D, rows, p.c.Hkv, 1)) != ACEFA_OK) {
            return rc;
        }
        if (rows && overlaps_cache(*t, *cache)) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    if (!aligned(cu_rows, 4) || !aligned(pos, 4)) {
        return ACEFA_ERR_LAYOUT;
    }
    DeviceCtx ctx;
    if ((rc = device_ctx(&ctx)) != ACEFA_OK) {
        return rc;
    }
    if (rows == 0) {
        note_launches(0, 0);
        return ACEFA_OK;
    }
    p.k_new = rows_of(*k_new), p.v_new = rows_of(*v_new);
    p.rows    = rows;
    p.cu      = cu_rows;
    p.per_set = (int) (rows / p.c.B);
    p.pos     = pos;
    p.dev_err = ctx.dev_err;
    if (launch_kv8_store(p, static_cast<cudaStream_t>(stream)) != cudaSuccess) {
        return ACEFA_ERR_CUDA;
    }
    note_launches(1, 0);
    return ACEFA_OK;
}

ACEFA_API int acefa_kv8_load(const acefa_kv8_cache *cache, const int32_t *len, const acefa_tensor *k_dst,
                             const acefa_tensor *v_dst, void *stream) {
    Kv8LoadParams p;
    std::memset(&p, 0, sizeof(p));
    if (!len || !k_dst || !v_dst || !k_dst->data || !v_dst->data) {
        return ACEFA_ERR_NULL;
    }
    int rc = check_cache(cache, false, &p.c);
    if (rc != ACEFA_OK) {
        return rc;
    }
    if (v_dst->type != k_dst->type) {
        return ACEFA_ERR_TYPE;
    }
    const int64_t n = k_dst->ne[1];
    if (n < 1 || n > p.c.n_max) {
        return ACEFA_ERR_SHAPE;
    }
    for (const acefa_tensor *t : {k_dst, v_dst}) {
        if ((rc = check_rows(*t, p.c.D, n, p.c.Hkv, p.c.B)) != ACEFA_OK) {
            return rc;
        }
        if (!disjoint(*t) || overlaps_cache(*t, *cache)) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    if (overlap(*k_dst, *v_dst) || !aligned(len, 4)) {
        return ACEFA_ERR_LAYOUT;
    }
    DeviceCtx ctx;
    if ((rc = device_ctx(&ctx)) != ACEFA_OK) {
        return rc;
    }
    p.k = rows_of(*k_dst), p.v = rows_of(*v_dst);
    p.n   = (int) n;
    p.len = len;
    if (launch_kv8_load(p, static_cast<cudaStream_t>(stream)) != cudaSuccess) {
        return ACEFA_ERR_CUDA;
    }
    note_launches(1, 0);
    return ACEFA_OK;
}

ACEFA_API size_t acefa_kv8_attn_workspace_bytes(const acefa_tensor *q, const acefa_kv8_cache *cache,
                                                const acefa_tensor *weight) {
    AttnPlan plan;
    return plan_attn(q, cache, weight, &plan) == ACEFA_OK ? plan.ws_bytes : 0;
}

ACEFA_API int acefa_kv8_attn(const acefa_tensor *q, const acefa_kv8_cache *cache, const int32_t *len,
                             const acefa_tensor *dst, float scale, const acefa_tensor *weight, void *stream,
                             void *workspace, size_t workspace_bytes) {
    if (!len || !dst || !dst->data) {
        return ACEFA_ERR_NULL;
    }
    AttnPlan  plan;
    const int plan_rc = plan_attn(q, cache, weight, &plan);
    if (plan_rc != ACEFA_OK && plan_rc != ACEFA_ERR_DEVICE && plan_rc != ACEFA_ERR_CUDA) {
        return plan_rc;
    }
    Kv8AttnParams &p  = plan.p;
    const int      rc = check_rows(*dst, p.c.D, q->ne[2], q->ne[1], p.c.B);
    if (rc != ACEFA_OK) {
        return rc;
    }
    if (!disjoint(*dst) || !aligned(len, 4) || overlap(*dst, *q) || overlaps_cache(*dst, *cache) ||
        (weight && (overlap(*dst, *weight) || overlap(*weight, *q) || overlaps_cache(*weight, *cache)))) {
        return ACEFA_ERR_LAYOUT;
    }
    if (!std::isfinite(scale)) {
        return ACEFA_ERR_SHAPE;
    }
    if (plan_rc != ACEFA_OK) {
        return plan_rc;
    }
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < plan.ws_bytes) {
        return ACEFA_ERR_WORKSPACE;
    }
    p.dst        = rows_of(*dst);
    p.len        = len;
    p.scale_log2 = scale * kLog2e;
    p.part       = static_cast<float *>(workspace);
    p.scores     = weight ? reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.part_bytes) : nullptr;
    const int launched = launch_kv8_attn(p, static_cast<cudaStream_t>(stream));
    if (launched == ACEFA_OK) {
        note_launches(p.cluster ? 1 : 2, 4);
    }
    return launched;
}

ACEFA_API int acefa_kv8_evict(const acefa_kv8_cache *cache, const acefa_tensor *weight, const int32_t *len,
                              int64_t n_first, int64_t n_recent, const acefa_kv8_cache *out,
                              const acefa_tensor *kept, const acefa_tensor *weight_out, int32_t *len_out,
                              void *stream) {
    Kv8EvictParams p;
    std::memset(&p, 0, sizeof(p));
    if (!weight || !weight->data || !len || !kept || !kept->data || !len_out || (weight_out && !weight_out->data)) {
        return ACEFA_ERR_NULL;
    }
    int rc = check_cache(cache, false, &p.c);
    if (rc == ACEFA_OK) {
        rc = check_cache(out, true, &p.out);
    }
    if (rc == ACEFA_OK) {
        rc = check_per_row(*weight, ACEFA_TYPE_F32, p.c.n_max, p.c, false);
    }
    if (rc != ACEFA_OK) {
        return rc;
    }
    const int64_t keep = kept->ne[0];
    if (p.out.D != p.c.D || p.out.Hkv != p.c.Hkv || p.out.B != p.c.B || keep < 1 || keep > p.out.n_max || n_first < 0 ||
        n_recent < 0 || n_first > keep || n_recent > keep - n_first) {
        return ACEFA_ERR_SHAPE;
    }
    if ((rc = check_per_row(*kept, ACEFA_TYPE_I32, keep, p.c, true)) != ACEFA_OK ||
        (weight_out && (rc = check_per_row(*weight_out, ACEFA_TYPE_F32, keep, p.c, true)) != ACEFA_OK)) {
        return rc;
    }
    const acefa_tensor *outs[6] = {&out->k, &out->v, &out->k_scale, &out->v_scale, kept, weight_out};
    for (int i = 0; i < 6; ++i) {
        if (!outs[i]) {
            continue;
        }
        if (overlaps_cache(*outs[i], *cache) || overlap(*outs[i], *weight) ||
            (i >= 4 && overlaps_cache(*outs[i], *out)) || (i == 5 && overlap(*weight_out, *kept))) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    if (!aligned(len, 4) || !aligned(len_out, 4)) {
        return ACEFA_ERR_LAYOUT;
    }
    {  // len may not be the array that len_out replaces: the heads' blocks read it at their own times
        const auto a = reinterpret_cast<uintptr_t>(len), b = reinterpret_cast<uintptr_t>(len_out);
        const auto n = (uintptr_t) p.c.B * sizeof(int32_t);
        if (a < b + n && b < a + n) {
            return ACEFA_ERR_LAYOUT;
        }
    }
    DeviceCtx ctx;
    if ((rc = device_ctx(&ctx)) != ACEFA_OK) {
        return rc;
    }
    p.weight = static_cast<const char *>(weight->data);
    p.w_nb2 = (int64_t) weight->nb[1], p.w_nb3 = (int64_t) weight->nb[2];
    p.len     = len;
    p.n_first = (int) n_first, p.n_recent = (int) n_recent, p.keep = (int) keep;
    p.kept  = static_cast<char *>(kept->data);
    p.k_nb2 = (int64_t) kept->nb[1], p.k_nb3 = (int64_t) kept->nb[2];
    if (weight_out) {
        p.weight_out = static_cast<char *>(weight_out->data);
        p.wo_nb2 = (int64_t) weight_out->nb[1], p.wo_nb3 = (int64_t) weight_out->nb[2];
    }
    p.len_out = len_out;
    if (launch_kv8_evict(p, static_cast<cudaStream_t>(stream)) != cudaSuccess) {
        return ACEFA_ERR_CUDA;
    }
    note_launches(2, 0);
    return ACEFA_OK;
}

}  // extern "C"
