// kv8_evict.cu -- eviction from the 8-bit block-scaled KV cache by accumulated
// attention weight (acefa_kv8_evict): a selection per (head, set), then a move.
//
// Selection.  A weight becomes a 32-bit key that orders like it; the keep-th
// largest key is found by a radix descent (11 + 11 + 10 bits, one histogram
// each, counts only, so atomics change nothing), and a scan in row order
// writes the rows above it and the first of those equal to it.  One CTA per
// (head, set); the weights are a few hundred KB that stay in L2.
// Move.  One CTA per 64 destination rows of (head, set) of K or V: it reads the
// rows' source blocks' scales, takes the largest, and copies the rows, rounding
// those of another scale once more.  Every source row and destination byte is
// touched once: HBM-bound, 2 bytes per value kept.
#include "kv8_internal.h"
#include "ptx.cuh"

namespace acefa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kBins       = 2048;
constexpr int kMoveThreads = 256;

// Orders like the weight: larger weight, larger key; -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) {
        return 0u;
    }
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 + 0 = 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) kv8_select_kernel(const __grid_constant__ Kv8EvictParams P) {
    __shared__ int      hist[kBins];
    __shared__ int      s_warp[2][kSelThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int      s_need;
    const int    h = blockIdx.x, b = blockIdx.y;
    const int    tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int    len  = clamp_len(__ldg(P.len + b), P.c.n_max);
    const int    kept = min(len, P.keep);
    const float *w    = reinterpret_cast<const float *>(P.weight + h * P.w_nb2 + b * P.w_nb3);
    int32_t     *out  = reinterpret_cast<int32_t *>(P.kept + h * P.k_nb2 + b * P.k_nb3);
    float *wo = P.weight_out ? reinterpret_cast<float *>(P.weight_out + h * P.wo_nb2 + b * P.wo_nb3) : nullptr;
    if (h == 0 && tid == 0) {
        P.len_out[b] = kept;
    }
    for (int x = kept + tid; x < P.keep; x += kSelThreads) {
        out[x] = -1;
        if (wo) {
            wo[x] = 0.0f;
        }
    }
    if (len <= P.keep) {
        for (int x = tid; x < len; x += kSelThreads) {
            out[x] = x;
            if (wo) {
                wo[x] = w[x];
            }
        }
        return;
    }
    // candidates: rows [lo, hi); the others stay.  len > keep >= n_first + n_recent.
    const int lo = P.n_first, hi = len - P.n_recent;
    if (tid == 0) {
        s_prefix = 0u;
        s_need   = P.keep - P.n_first - P.n_recent;  // of the candidates
    }
    // ---- the need-th largest key, and how many of those equal to it are kept
    const int shifts[3] = {21, 10, 0};
    uint32_t  mask      = 0u;  // bits of the key settled so far
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = shifts[pass], bins = pass == 2 ? 1024 : 2048;
        for (int x = tid; x < kBins; x += kSelThreads) {
            hist[x] = 0;
        }
        __syncthreads();
        const uint32_t prefix = s_prefix;
        const int      need   = s_need;
        if (need == 0) {
            break;  // uniform
        }
        for (int x0 = lo + warp * 32; x0 < hi; x0 += kSelThreads) {
            const int      x   = x0 + lane;
            const uint32_t key = x < hi ? order_key(__ldg(w + x)) : 0u;
            const bool     on  = x < hi && (key & mask) == prefix;
            const int      bin = on ? (int) ((key >> shift) & (uint32_t) (bins - 1)) : -1;
            const unsigned eq  = __match_any_sync(0xffffffffu, bin);  // many weights share a bin (zeros)
            if (on && lane == __ffs(eq) - 1) {
                atomicAdd(&hist[bin], __popc(eq));
            }
        }
        __syncthreads();
        // suffix sums from the largest bin; the bin where they reach `need`
        const int b0 = kBins - 2 - 2 * tid;  // this thread: bins b0 + 1, b0, from the top
        const int c1 = hist[b0 + 1], c0 = hist[b0];
        int       incl = c1 + c0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            incl += lane >= off ? v : 0;
        }
        if (lane == 31) {
            s_warp[0][warp] = incl;
        }
        __syncthreads();
        int before = 0;
        for (int k = 0; k < warp; ++k) {
            before += s_warp[0][k];
        }
        const int above1 = before + incl - c1 - c0;  // keys in bins above b0 + 1
        const int above0 = above1 + c1;
        if (above1 < need && need <= above1 + c1) {
            s_prefix = prefix | (uint32_t) (b0 + 1) << shift;
            s_need   = need - above1;
        } else if (above0 < need && need <= above0 + c0) {
            s_prefix = prefix | (uint32_t) b0 << shift;
            s_need   = need - above0;
        }
        mask |= (uint32_t) (bins - 1) << shift;
        __syncthreads();
    }
    const uint32_t top  = s_prefix;
    const int      need = s_need;                              // rows equal to `top` that stay, 0: none at all
    const bool     none = P.keep == P.n_first + P.n_recent;    // no candidate stays
    // ---- rows in order: each thread owns a contiguous run
    const int per = (len + kSelThreads - 1) / kSelThreads;
    const int r0 = min(len, tid * per), r1 = min(len, r0 + per);
    int       n_eq = 0, n_sure = 0;
    for (int x = r0; x < r1; ++x) {
        if (x < lo || x >= hi) {
            ++n_sure;
        } else if (!none) {
            const uint32_t key = order_key(__ldg(w + x));
            n_eq += key == top;
            n_sure += key > top;
        }
    }
    int i_eq = n_eq, i_sure = n_sure;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, i_eq, off), v = __shfl_up_sync(0xffffffffu, i_sure, off);
        i_eq += lane >= off ? u : 0;
        i_sure += lane >= off ? v : 0;
    }
    if (lane == 31) {
        s_warp[0][warp] = i_eq;
        s_warp[1][warp] = i_sure;
    }
    __syncthreads();
    for (int k = 0; k < warp; ++k) {
        i_eq += s_warp[0][k];
        i_sure += s_warp[1][k];
    }
    int eq = i_eq - n_eq;                            // equal rows before this run
    int at = i_sure - n_sure + min(eq, none ? 0 : need);  // kept rows before it
    for (int x = r0; x < r1; ++x) {
        bool stay = x < lo || x >= hi;
        if (!stay && !none) {
            const uint32_t key = order_key(__ldg(w + x));
            stay               = key > top || (key == top && eq < need);
            eq += key == top;
        }
        if (stay) {
            out[at] = x;
            if (wo) {
                wo[at] = w[x];
            }
            ++at;
        }
    }
}

// grid (64-row blocks of `keep`, Hkv, 2 * B)
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv8_move_kernel(const __grid_constant__ Kv8EvictParams P) {
    constexpr int kLanes = D / 4;
    constexpr int kRows  = kMoveThreads / kLanes;
    constexpr int kPass  = kKv8Block / kRows;
    __shared__ int   s_row[kKv8Block];
    __shared__ float s_d[kKv8Block];
    __shared__ float s_top[2];
    const int      blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z >> 1;
    const Kv8Side &src = (blockIdx.z & 1) ? P.c.v : P.c.k;
    const Kv8Side &dst = (blockIdx.z & 1) ? P.out.v : P.out.k;
    const int      lo  = blk * kKv8Block;
    const int      n   = min(kKv8Block, P.keep - lo);  // rows of the block that are written
    const int32_t *kept = reinterpret_cast<const int32_t *>(P.kept + h * P.k_nb2 + b * P.k_nb3);
    pdl_wait_primary();
    if (threadIdx.x < kKv8Block) {
        const int x = threadIdx.x;
        // written by the selection; a value that is no row moves nothing
        const int   row = x < n ? __ldcg(kept + lo + x) : -1;
        const bool  on  = row >= 0 && row < P.c.n_max;
        const float d   = on ? *(reinterpret_cast<const float *>(reinterpret_cast<const char *>(src.scale) +
                                                               h * src.s_nb2 + b * src.s_nb3) +
                               row / kKv8Block)
                             : 0.0f;
        s_row[x] = on ? row : -1;
        s_d[x]   = d;
        float top = d;
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
        }
        if ((x & 31) == 0) {
            s_top[x >> 5] = top;
        }
    }
    __syncthreads();
    const float    d_new = max_nan(s_top[0], s_top[1]);
    const int      r0 = threadIdx.x / kLanes, e0 = 4 * (threadIdx.x % kLanes);
    const int8_t  *sp = src.q + h * src.nb2 + b * src.nb3;
    int8_t        *dp = dst.q + (int64_t) lo * dst.nb1 + h * dst.nb2 + b * dst.nb3;
    uint32_t       w[kPass];
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int row = s_row[r0 + p * kRows];
        w[p]          = row >= 0 ? __ldcs(reinterpret_cast<const uint32_t *>(sp + (int64_t) row * src.nb1 + e0)) : 0u;
    }
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int   r = r0 + p * kRows;
        const float d = s_d[r];
        if (d != d_new && w[p]) {
            w[p] = requant4(w[p], d, d_new, __fdiv_rn(d, d_new));
        }
        if (r < n) {
            *reinterpret_cast<uint32_t *>(dp + (int64_t) r * dst.nb1 + e0) = w[p];
        }
    }
    if (threadIdx.x == 0) {
        *(reinterpret_cast<float *>(reinterpret_cast<char *>(dst.scale) + h * dst.s_nb2 + b * dst.s_nb3) + blk) = d_new;
    }
}

}  // namespace

cudaError_t launch_kv8_evict(const Kv8EvictParams &p, cudaStream_t s) {
    kv8_select_kernel<<<dim3((unsigned) p.c.Hkv, (unsigned) p.c.B), kSelThreads, 0, s>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        return e;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3((unsigned) ((p.keep + kKv8Block - 1) / kKv8Block), (unsigned) p.c.Hkv,
                                  (unsigned) (2 * p.c.B));
    cfg.blockDim           = dim3(kMoveThreads);
    cfg.stream             = s;
    cfg.attrs              = attr;
    cfg.numAttrs           = 1;
    return p.c.D == 128 ? cudaLaunchKernelEx(&cfg, kv8_move_kernel<128>, p)
                        : cudaLaunchKernelEx(&cfg, kv8_move_kernel<64>, p);
}

}  // namespace acefa
