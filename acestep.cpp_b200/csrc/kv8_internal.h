// kv8_internal.h -- parameter blocks and device helpers shared by the kernels
// of the 8-bit block-scaled KV cache (acefa_kv8_*).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fa_internal.h"
#include "ptx.cuh"

namespace acefa {

constexpr int kKv8Block   = ACEFA_KV8_BLOCK;     // tokens that share a scale
constexpr int kKv8MaxSets = ACEFA_KV8_MAX_SETS;  // sets of a cache

// One of K and V of a cache, after validation.  Strides in bytes.
struct Kv8Side {
    int8_t *q;      // rows of D values
    float  *scale;  // one per block
    int64_t nb1, nb2, nb3;    // row, head, set
    int64_t s_nb2, s_nb3;     // scales: head, set (blocks are contiguous)
};
struct Kv8Dev {
    Kv8Side k, v;
    int     D, n_max, Hkv, B;
};

// An F32 / F16 / BF16 tensor [D, rows, H, B] read or written by the kernels.
struct Kv8Rows {
    char   *data;
    int64_t nb1, nb2, nb3;
    int     type;
};

struct Kv8StoreParams {
    Kv8Dev         c;
    Kv8Rows        k_new, v_new;  // nb3 unused
    int64_t        rows;          // rows of k_new (at most 2^30)
    const int32_t *cu;            // or nullptr: per_set rows each
    int            per_set;
    const int32_t *pos;
    int           *dev_err;
};
struct Kv8LoadParams {
    Kv8Dev         c;
    Kv8Rows        k, v;
    int            n;  // rows of the destination
    const int32_t *len;
};
struct Kv8AttnParams {
    Kv8Dev         c;
    Kv8Rows        q, dst;  // q: nb1 = query, nb2 = head; dst: nb1 = head, nb2 = query
    const int32_t *len;
    char          *weight;  // F32 [n_max, Hkv, B] or nullptr
    int64_t        w_nb2, w_nb3;
    int            n_q, G, rows;  // rows = G * n_q per kv head
    int            n_rb;          // row blocks per (set, kv head)
    int            n_cta;         // CTAs of the split kernel
    int            cluster;       // CTAs of a unit's cluster, or 0: the split kernel and the sum kernel
    float          scale_log2;    // scale * log2(e)
    float         *part;          // partial results, one slot per (CTA, unit) that meet
    float         *scores;        // [unit][n_max][score_stride] log2-unit scores, with weights only
    int            score_stride;
    int           *dev_err;
    uint64_t       wait_limit_ns;
};
struct Kv8EvictParams {
    Kv8Dev         c, out;
    const char    *weight;  // F32 [n_max, Hkv, B]
    int64_t        w_nb2, w_nb3;
    const int32_t *len;
    int            n_first, n_recent, keep;
    char          *kept;  // I32 [keep, Hkv, B]
    int64_t        k_nb2, k_nb3;
    char          *weight_out;  // F32 or nullptr
    int64_t        wo_nb2, wo_nb3;
    int32_t       *len_out;
};

cudaError_t launch_kv8_store(const Kv8StoreParams &p, cudaStream_t s);
cudaError_t launch_kv8_load(const Kv8LoadParams &p, cudaStream_t s);
int         launch_kv8_attn(const Kv8AttnParams &p, cudaStream_t s);  // acefa_status
cudaError_t launch_kv8_evict(const Kv8EvictParams &p, cudaStream_t s);

// Rows of a unit of the attention kernel and the CTAs that it may keep
// resident on one SM; functions of the operands alone.  More than eight F32
// rows go in units of eight that read the keys again (from L2): split Q
// fragments of sixteen rows do not fit the registers of two CTAs per SM.  The
// output's type is not known where the workspace is sized, so 16-bit rows with an
// F32 output, which split too, stay in units of sixteen and spill (4 sets of 8192 rows,
// 8 heads of 16 rows, D = 128: 36 us, from F32 rows 30, with a 16-bit output 23).
inline int kv8_unit_rows(int rows, int q_type) { return rows <= 8 || q_type == ACEFA_TYPE_F32 ? 8 : 16; }
int        kv8_attn_ctas_per_sm();
int        kv8_attn_cluster(const Kv8AttnParams &p, int64_t units, int sm_count);
inline size_t kv8_slot_floats(int D, int unit_rows) { return (size_t) unit_rows * (D + 2); }

// ------------------------------------------------------------------ device helpers
#ifdef __CUDACC__

// Launches a kernel that begins with pdl_wait_primary(): its blocks are set up
// while the stream's previous kernel ends, and wait there until it has.  What they
// read may still be written while they wait, so no load of theirs may go the
// read-only way (__ldg), which wants data that is constant from the kernel's start.  One
// exception reads before its wait: kv8_attn_sum_kernel takes the lengths, which the kernel
// ahead of it (kv8_attn_kernel, which lets it start) has waited for.  Measured,
// back to back: 0.2 us of a call of few rows, 0.3 of a store and of an eviction's
// kernels each.  (Letting the next kernel start earlier, behind that wait, cost time:
// store + load of one token 4.6 -> 5.2 us, eviction 15.7 -> 16.7, packed prompts 78 -> 81.)
template <class... K, class... A>
cudaError_t launch_pdl(void (*kernel)(K...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A &...args) {
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = grid;
    cfg.blockDim           = dim3((unsigned) threads);
    cfg.dynamicSmemBytes   = smem;
    cfg.stream             = s;
    cfg.attrs              = attr;
    cfg.numAttrs           = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Finds item x among the items of n segments, count(i) of segment i in their
// order (fewer than 2^31 in all); a negative count ends them.  The whole warp calls
// it with the same arguments and gets the same answer: the segment and the item's
// number in it, or false behind the last.
template <class F>
__device__ __forceinline__ bool find_item(int n, int x, F count, int &seg, int &item) {
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < n; base += 32) {
        int            mine = base + lane < n ? count(base + lane) : 0;
        const unsigned end  = __ballot_sync(0xffffffffu, mine < 0);
        mine                = end && lane >= __ffs(end) - 1 ? 0 : mine;
        int incl            = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            incl += lane >= off ? v : 0;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, x < incl);
        if (hit) {
            const int l = __ffs(hit) - 1;
            seg         = base + l;
            item        = x - __shfl_sync(0xffffffffu, incl - mine, l);
            return true;
        }
        if (end) {
            return false;
        }
        x -= __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

__device__ __forceinline__ int clamp_len(int len, int n_max) { return len < 0 ? 0 : (len > n_max ? n_max : len); }

// max that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); }

// x / d rounded to the nearest integer, ties to even, as if the quotient were
// exact, clamped to 127.  Rounding is monotonic, so rounding the F32 quotient
// t can only differ where t landed on a half-integer h; there the sign of
// x - h * d (one FMA: h * d is exact inside it) says on which side of h the
// true quotient lies.  d > 0 and finite; the result is 0 for d == 0 and NaN.
__device__ __forceinline__ int quant_rne(float x, float d) {
    const float t = __fdiv_rn(x, d);
    float       q = rintf(t);
    if (fabsf(t - truncf(t)) == 0.5f) {
        const float r = fmaf(-t, d, x);
        if (r != 0.0f) {
            q = r > 0.0f ? ceilf(t) : floorf(t);
        }
    }
    q = fminf(fmaxf(q, -127.0f), 127.0f);
    return d > 0.0f ? __float2int_rn(q) : 0;  // NaN converts to 0
}

// q * d_old / d_new rounded once to the nearest integer, ties to even, for
// |q| <= 127 and d_old <= d_new: q * d_old is exact in F64 and the division
// rounds correctly (a tie is then a tie, and nothing else is within 2^-40 of one).
__device__ __forceinline__ int requant_rne(int q, float d_old, float d_new) {
    return d_new > 0.0f ? (int) rint(__ddiv_rn((double) q * (double) d_old, (double) d_new)) : 0;
}

// Adding 1.5 * 2^23 rounds an F32 number below 2^22 to an integer (ties to even)
// that stands in the low bits of the sum.
constexpr float kRoundMagic = 12582912.0f;
// How near a half-integer v * f, taken for the true quotient, may not be: with
// f in error by 2^-23 (a rounded reciprocal or ratio) and |v * f| <= 127 the
// quotient is within 2^-15 of it, and beyond that distance both round alike.
constexpr float kNearTie = 0.5f - 3.0517578125e-5f;

// The low bytes of four rounded sums.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040u),
                       __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040u), 0x5410u);
}

// Four values of a block of scale d; inv = 1 / d rounded, or 0 where the quick
// way does not hold (d = 0, subnormal or not a number).
__device__ __forceinline__ uint32_t quant4(float4 x, float d, float inv) {
    const uint64_t v[2] = {f32x2(x.x, x.y), f32x2(x.z, x.w)}, i2 = f32x2(inv, inv);
    const uint64_t magic = f32x2(kRoundMagic, kRoundMagic), minus = f32x2(-1.0f, -1.0f);
    float          y[4], off = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // two values per instruction
        const uint64_t s = ffma2(v[e], i2, magic);
        float          d0, d1;
        f32x2_split(ffma2(v[e], i2, ffma2(s, minus, magic)), d0, d1);
        f32x2_split(s, y[2 * e], y[2 * e + 1]);
        off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
    }
    if (off < kNearTie && inv != 0.0f) {
        return low_bytes(y[0], y[1], y[2], y[3]);
    }
    return (uint32_t) (quant_rne(x.x, d) & 0xFF) | (uint32_t) (quant_rne(x.y, d) & 0xFF) << 8 |
           (uint32_t) (quant_rne(x.z, d) & 0xFF) << 16 | (uint32_t) (quant_rne(x.w, d) & 0xFF) << 24;
}
// 1 / d for quant4
__device__ __forceinline__ float quant_inv(float d) { return d >= 1.1754944e-36f && d <= 1.0e36f ? __frcp_rn(d) : 0.0f; }

// Four int8 values of a 32-bit word moved from scale d_old to d_new, ratio =
// d_old / d_new rounded.
__device__ __forceinline__ uint32_t requant4(uint32_t w, float d_old, float d_new, float ratio) {
    const uint32_t b = w ^ 0x80808080u;  // int8 + 128
    const uint64_t bias = f32x2(-8388736.0f, -8388736.0f), r2 = f32x2(ratio, ratio);
    const uint64_t magic = f32x2(kRoundMagic, kRoundMagic), minus = f32x2(-1.0f, -1.0f);
    float          y[4], off = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e += 2) {  // two values per instruction
        // 2^23 + byte, exactly
        const uint64_t q = fadd2(f32x2(__uint_as_float(__byte_perm(b, 0x4B000000u, 0x7650u + (uint32_t) e)),
                                       __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7651u + (uint32_t) e))),
                                 bias);
        const uint64_t s = ffma2(q, r2, magic);
        float          d0, d1;
        f32x2_split(ffma2(q, r2, ffma2(s, minus, magic)), d0, d1);
        f32x2_split(s, y[e], y[e + 1]);
        off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
    }
    if (off < kNearTie) {
        return low_bytes(y[0], y[1], y[2], y[3]);
    }
    uint32_t o = 0;
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
        o |= (uint32_t) (requant_rne((int) (int8_t) (w >> (8 * e)), d_old, d_new) & 0xFF) << (8 * e);
    }
    return o;
}

// Four consecutive values of a row of type T at element e0, as F32.
template <class T>
__device__ __forceinline__ float4 load4(const char *row, int e0, bool vec) {
    const T *p = reinterpret_cast<const T *>(row) + e0;
    if constexpr (sizeof(T) == 4) {
        return vec ? __ldcs(reinterpret_cast<const float4 *>(p)) : make_float4(p[0], p[1], p[2], p[3]);
    } else {
        alignas(8) T v[4];
        if (vec) {
            *reinterpret_cast<uint2 *>(v) = __ldcs(reinterpret_cast<const uint2 *>(p));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = p[e];
            }
        }
        return make_float4((float) v[0], (float) v[1], (float) v[2], (float) v[3]);
    }
}
template <class T>
__device__ __forceinline__ void store4(char *row, int e0, float4 x, bool vec) {
    T *p = reinterpret_cast<T *>(row) + e0;
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            __stcs(reinterpret_cast<float4 *>(p), x);
        } else {
            p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
        }
    } else {
        alignas(8) T v[4] = {(T) x.x, (T) x.y, (T) x.z, (T) x.w};
        if (vec) {
            __stcs(reinterpret_cast<uint2 *>(p), *reinterpret_cast<uint2 *>(v));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = v[e];
            }
        }
    }
}

#endif  // __CUDACC__

}  // namespace acefa
