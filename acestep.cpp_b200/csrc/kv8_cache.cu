// kv8_cache.cu -- writing and reading the 8-bit block-scaled KV cache
// (acefa_kv8_store, acefa_kv8_load).
//
// A block is 64 rows of one (head, set) of K or V; its rows share the scale
// d = amax / 127, so a block can only be quantised once all of its new rows
// have been seen.  The store kernel gives each block it touches to one CTA,
// which holds the block's new rows in registers (32 values per thread) between
// the maximum and the rounding: every input is read once and every byte
// written once.  Rows that were in the block before stay as they are unless
// the block's scale has to grow; only then are they read and rounded again.
// Both kernels stream: 4 + 1 bytes per value stored from F32, 1 + 4 loaded to
// F32, with 16 B or 4 B per lane and whole lines per warp.  Measured (B200): 8086
// rows x 8 heads x 128 of K and V from F32 stored in 18-21 us (4.0-4.6 TB/s, bound by
// instruction issue, 62 %), 16384 rows read back in 22.5 us (7.4 TB/s); both together
// 40.9 us with 256 threads per block of rows (128: 42.5, 512: 48.6 against 40.7 then).
#include "kv8_internal.h"
#include "ptx.cuh"

namespace acefa {
namespace {

constexpr int kThreads = 256;

// Rows of set s among k_new (first row, count), the cache row of the first, and
// whether they are none (count 0).  All fit in 32 bits.
struct SetRows {
    int  first, count, pos;
    bool bad;
};
__device__ __forceinline__ SetRows set_rows(const Kv8StoreParams &P, int s) {
    SetRows r;
    r.pos = P.pos[s];
    if (P.cu) {
        r.first         = P.cu[s];
        const int end   = P.cu[s + 1];
        r.bad           = r.first < 0 || end < r.first || end > (int) P.rows;
        r.count         = r.bad ? 0 : end - r.first;
    } else {
        r.count = P.per_set;
        r.first = r.count * s;
        r.bad   = false;
    }
    if (r.count > 0 && (r.pos < 0 || r.pos > P.c.n_max - r.count)) {
        r.bad   = true;
        r.count = 0;
    }
    return r;
}
__device__ __forceinline__ int blocks_of(const SetRows &r) {
    return r.count > 0 ? (r.pos + r.count - 1) / kKv8Block - r.pos / kKv8Block + 1 : 0;
}

// grid (blocks touched, an upper bound; Hkv; K and V).  A thread holds four
// values of a row (T = its source type) and D / 4 threads a row.
template <int D, class T>
__global__ void __launch_bounds__(kThreads) kv8_store_kernel(const __grid_constant__ Kv8StoreParams P) {
    constexpr int kLanes = D / 4;               // threads per row
    constexpr int kRows  = kThreads / kLanes;   // rows per pass
    constexpr int kPass  = kKv8Block / kRows;   // passes over the block
    __shared__ uint32_t s_max[kThreads / 32];
    pdl_wait_primary();
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
        for (int s = threadIdx.x; s < P.c.B; s += kThreads) {
            if (set_rows(P, s).bad) {
                atomicCAS(P.dev_err, 0, DEVERR_APPEND_POS);
            }
        }
    }
    int s, item;
    if (!find_item(P.c.B, blockIdx.x, [&](int i) { return blocks_of(set_rows(P, i)); }, s, item)) {
        return;
    }
    const SetRows  rows = set_rows(P, s);
    const int      pos  = rows.pos;
    const int      h    = blockIdx.y;
    const Kv8Rows &src  = blockIdx.z ? P.v_new : P.k_new;
    const Kv8Side &side = blockIdx.z ? P.c.v : P.c.k;
    const int      blk  = pos / kKv8Block + item;
    const int      lo   = blk * kKv8Block;                                        // first row of the block
    const int      a    = max(lo, pos);                                           // first new row
    const int      hi   = min(lo + kKv8Block, pos + rows.count);                  // behind the last one
    const int      r0   = threadIdx.x / kLanes, e0 = 4 * (threadIdx.x % kLanes);
    const char    *base = src.data + (rows.first + (a - pos)) * src.nb1 + h * src.nb2;
    const bool     vec  = ((reinterpret_cast<uintptr_t>(base) | (uintptr_t) src.nb1) & (4 * sizeof(T) - 1)) == 0;
    float4         x[kPass];
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int r = lo + r0 + p * kRows;
        x[p]        = r >= a && r < hi ? load4<T>(base + (int64_t) (r - a) * src.nb1, e0, vec)
                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float  *scale = reinterpret_cast<float *>(reinterpret_cast<char *>(side.scale) + h * side.s_nb2 + s * side.s_nb3) +
                   blk;
    const float d_old = a > lo ? *scale : 0.0f;
    float most = 0.0f;  // of |x|, or a NaN
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        most = fmax3_nan(most, fabsf(x[p].x), fabsf(x[p].y));
        most = fmax3_nan(most, fabsf(x[p].z), fabsf(x[p].w));
    }
    // as bits: they order like |x|, infinities and NaNs above all
    uint32_t top = __float_as_uint(most) & 0x7FFFFFFFu;
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) {
        s_max[threadIdx.x >> 5] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        top = max(top, s_max[w]);
    }
    const float d = top >= 0x7F800000u ? NAN : max_nan(__fdiv_rn(__uint_as_float(top), 127.0f), d_old);
    const float inv = quant_inv(d);
    int8_t     *qb = side.q + (int64_t) lo * side.nb1 + h * side.nb2 + s * side.nb3;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int r = r0 + p * kRows;
        if (lo + r >= a && lo + r < hi) {
            *reinterpret_cast<uint32_t *>(qb + r * side.nb1 + e0) = quant4(x[p], d, inv);
        }
    }
    if (a > lo && d > d_old) {  // the rows that stay move to the new scale
        const float ratio = __fdiv_rn(d_old, d);
        for (int r = r0; lo + r < a; r += kRows) {
            uint32_t *w = reinterpret_cast<uint32_t *>(qb + (int64_t) r * side.nb1 + e0);
            *w          = requant4(*w, d_old, d, ratio);
        }
    }
    if (threadIdx.x == 0) {
        *scale = d;
    }
}

// grid (64-row blocks of the destination, Hkv, 2 * B)
template <int D, class T>
__global__ void __launch_bounds__(kThreads) kv8_load_kernel(const __grid_constant__ Kv8LoadParams P) {
    constexpr int  kLanes = D / 4;
    constexpr int  kRows  = kThreads / kLanes;
    constexpr int  kPass  = kKv8Block / kRows;
    pdl_wait_primary();
    const int      blk = blockIdx.x, h = blockIdx.y, s = blockIdx.z >> 1;
    const Kv8Rows &dst  = (blockIdx.z & 1) ? P.v : P.k;
    const Kv8Side &side = (blockIdx.z & 1) ? P.c.v : P.c.k;
    const int      len  = min(clamp_len(P.len[s], P.c.n_max), P.n);
    const int      lo   = blk * kKv8Block;
    const int      r0 = threadIdx.x / kLanes, e0 = 4 * (threadIdx.x % kLanes);
    const int8_t  *qb = side.q + (int64_t) lo * side.nb1 + h * side.nb2 + s * side.nb3;
    char          *out = dst.data + (int64_t) lo * dst.nb1 + h * dst.nb2 + s * dst.nb3;
    const bool     vec = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t) dst.nb1) & (4 * sizeof(T) - 1)) == 0;
    uint32_t       w[kPass];
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int r = r0 + p * kRows;
        w[p]        = lo + r < len ? __ldcs(reinterpret_cast<const uint32_t *>(qb + (int64_t) r * side.nb1 + e0)) : 0u;
    }
    const float d = lo < len ? *(reinterpret_cast<const float *>(reinterpret_cast<const char *>(side.scale) +
                                                                 h * side.s_nb2 + s * side.s_nb3) +
                                 blk)
                             : 0.0f;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int r = r0 + p * kRows;
        if (lo + r < P.n) {
            const bool  live = lo + r < len;  // (a NaN scale must not reach the zeros)
            const float f    = live ? d : 0.0f;
            store4<T>(out + (int64_t) r * dst.nb1, e0,
                      make_float4((float) (int8_t) w[p] * f, (float) (int8_t) (w[p] >> 8) * f,
                                  (float) (int8_t) (w[p] >> 16) * f, (float) (int8_t) (w[p] >> 24) * f),
                      vec);
        }
    }
}

template <class K, class P>
cudaError_t by_type(int D, int type, dim3 grid, cudaStream_t s, const P &p, K pick) {
    void (*k)(const P) = pick(D, type);
    return launch_pdl(k, grid, kThreads, 0, s, p);
}

}  // namespace

cudaError_t launch_kv8_store(const Kv8StoreParams &p, cudaStream_t s) {
    // a set of n rows touches at most (n + 62) / 64 + 1 blocks
    const int64_t per  = p.cu ? 0 : (p.rows / p.c.B + 62) / kKv8Block + 1;
    const int64_t most = p.cu ? p.rows / kKv8Block + 2 * (int64_t) p.c.B : per * p.c.B;
    dim3          grid((unsigned) most, (unsigned) p.c.Hkv, 2);
    return by_type(p.c.D, p.k_new.type, grid, s, p, [](int D, int type) {
        return D == 128 ? (type == ACEFA_TYPE_F32   ? kv8_store_kernel<128, float>
                           : type == ACEFA_TYPE_F16 ? kv8_store_kernel<128, __half>
                                                    : kv8_store_kernel<128, __nv_bfloat16>)
                        : (type == ACEFA_TYPE_F32   ? kv8_store_kernel<64, float>
                           : type == ACEFA_TYPE_F16 ? kv8_store_kernel<64, __half>
                                                    : kv8_store_kernel<64, __nv_bfloat16>);
    });
}

cudaError_t launch_kv8_load(const Kv8LoadParams &p, cudaStream_t s) {
    dim3 grid((unsigned) ((p.n + kKv8Block - 1) / kKv8Block), (unsigned) p.c.Hkv, (unsigned) (2 * p.c.B));
    return by_type(p.c.D, p.k.type, grid, s, p, [](int D, int type) {
        return D == 128 ? (type == ACEFA_TYPE_F32   ? kv8_load_kernel<128, float>
                           : type == ACEFA_TYPE_F16 ? kv8_load_kernel<128, __half>
                                                    : kv8_load_kernel<128, __nv_bfloat16>)
                        : (type == ACEFA_TYPE_F32   ? kv8_load_kernel<64, float>
                           : type == ACEFA_TYPE_F16 ? kv8_load_kernel<64, __half>
                                                    : kv8_load_kernel<64, __nv_bfloat16>);
    });
}

}  // namespace acefa
