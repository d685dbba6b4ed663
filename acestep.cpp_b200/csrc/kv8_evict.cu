// kv8_evict.cu -- eviction from the 8-bit block-scaled KV cache by accumulated
// attention weight (acefa_kv8_evict): a selection per (head, set), then a move.
//
// Selection.  A weight becomes a 32-bit key that orders like it; the keep-th
// largest key is found by a radix descent (11 + 11 + 10 bits, one histogram
// each, counts only, so the atomics' order changes nothing; it ends early where
// a whole bin stays), and a scan in row order writes the rows above it and
// the first of those equal to it.  One CTA per (head, set), the keys in registers
// up to 8192 rows (9 us for 64 CTAs of 8192 rows; from shared memory 13): bound by
// the latency of its passes.
// Move.  One CTA per 64 destination rows of K and V of a (head, set): it reads the
// rows' source blocks' scales, takes the largest, and copies the rows, rounding
// those of another scale once more.  Every source row and destination byte is
// touched once, 2 bytes per value kept.  Measured (B200), 8 sets x 8 heads, 8192
// rows to 4000: selection 9 us, move 25 us (5.2 TB/s); 2 sets, 2048 to 1024: 7 and 6 us.
#include "kv8_internal.h"
#include "ptx.cuh"

namespace acefa {
namespace {

constexpr int kSelThreads  = 1024;
constexpr int kSelWarps    = kSelThreads / 32;
constexpr int kBins        = 2048;
constexpr int kSelMaxKeys  = 49152;  // keys held in shared memory; more are read again from L2
constexpr int kSelRegs     = 8;      // of a thread: keys held in registers up to 8192 rows
constexpr int kShared = 0, kAgain = -1;
constexpr int kMoveThreads = 256;

// Orders like the weight: larger weight, larger key; -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) {
        return 0u;
    }
    const uint32_t b = __float_as_uint(w + 0.0f);  // -0 + 0 = 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One CTA per (head, set); each warp owns a run of consecutive rows and a thread
// every 32nd of them.  Where its keys wait between the passes: K > 0, in K
// registers (up to 1024 K rows); kShared, in shared memory; kAgain, read again from L2
// (32768 rows: 24 us from shared memory, 29 us from L2).
template <int K>
__global__ void __launch_bounds__(kSelThreads, 1) kv8_select_kernel(const __grid_constant__ Kv8EvictParams P) {
    extern __shared__ uint32_t s_key[];
    __shared__ int      s_hist[3][kBins];
    __shared__ int      s_eq[kSelWarps], s_sure[kSelWarps];
    __shared__ uint32_t s_prefix;
    __shared__ int      s_need, s_done;
    pdl_wait_primary();
    const int    h = blockIdx.x, b = blockIdx.y;
    const int    tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int    len  = clamp_len(P.len[b], P.c.n_max);
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
    const int  lo = P.n_first, hi = len - P.n_recent;
    const bool none = P.keep == P.n_first + P.n_recent;  // no candidate stays
    const int  steps = (len + kSelThreads - 1) / kSelThreads;  // rows of a thread, K at most
    const int  r0 = min(len, warp * steps * 32), r1 = min(len, r0 + steps * 32);  // the warp's run
    uint32_t   reg[K > 0 ? K : 1];
    if constexpr (K > 0) {
        float v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {  // all on their way together
            v[i] = r0 + 32 * i + lane < r1 ? w[r0 + 32 * i + lane] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < K; ++i) {
            reg[i] = order_key(v[i]);
        }
    } else if constexpr (K == kShared) {
        for (int x = r0 + lane; x < r1; x += 4 * 32) {  // four loads on their way
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = x + e * 32 < r1 ? w[x + e * 32] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (x + e * 32 < r1) {
                    s_key[x + e * 32] = order_key(v[e]);  // read by this thread alone
                }
            }
        }
    }
    // f(row, key) for the rows of this thread; rows at or past r1 are none.  All
    // threads take the same number of steps, so f may vote.
    auto each_row = [&](auto f) {
        if constexpr (K > 0) {
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if (i < steps) {
                    f(r0 + 32 * i + lane, reg[i]);
                }
            }
        } else {
#pragma unroll 4
            for (int i = 0; i < steps; ++i) {
                const int x = r0 + 32 * i + lane;
                f(x, x < r1 ? (K == kShared ? s_key[x] : order_key(w[x])) : 0u);
            }
        }
    };
    for (int x = tid; x < 3 * kBins; x += kSelThreads) {
        s_hist[0][x] = 0;
    }
    if (tid == 0) {
        s_prefix = 0u;
        s_need   = P.keep - P.n_first - P.n_recent;  // of the candidates
        s_done   = 0;
    }
    __syncthreads();
    // ---- the need-th largest key, and how many of those equal to it are kept
    const int shifts[3] = {21, 10, 0};
    uint32_t  mask      = 0u;  // bits of the key settled so far
#pragma unroll 1
    for (int pass = 0; pass < 3 && !none; ++pass) {
        const int      shift = shifts[pass], bins = pass == 2 ? 1024 : 2048;
        int           *hist   = s_hist[pass];
        const uint32_t prefix = s_prefix;
        const int      need   = s_need;
        each_row([&](int x, uint32_t key) {
            if (x >= lo && x < min(hi, r1) && (key & mask) == prefix) {
                atomicAdd(&hist[(key >> shift) & (uint32_t) (bins - 1)], 1);
            }
        });
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
            s_eq[warp] = incl;
        }
        __syncthreads();
        const int before = (int) __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0);
        const int above1 = before + incl - c1 - c0;  // keys in bins above b0 + 1
        const int above0 = above1 + c1;
        const bool in1 = above1 < need && need <= above1 + c1, in0 = above0 < need && need <= above0 + c0;
        if (in1 || in0) {
            const uint32_t bin  = (uint32_t) (in1 ? b0 + 1 : b0);
            const int      left = need - (in1 ? above1 : above0);
            if (left == (in1 ? c1 : c0)) {
                // the whole bin stays: everything above the key before its first
                s_done   = 1;
                s_prefix = prefix | bin << shift;
                s_need   = 0;
            } else {
                s_prefix = prefix | bin << shift;
                s_need   = left;
            }
        }
        mask |= (uint32_t) (bins - 1) << shift;
        __syncthreads();
        if (s_done) {
            break;  // uniform
        }
    }
    // a candidate stays with a key above `top`, or as one of the first `need` equal
    // to it.  (A bin that starts at key 0 and stays whole keeps every candidate:
    // len > keep rules that out, so top - 1 does not wrap.)
    const uint32_t top  = s_done ? s_prefix - 1u : s_prefix;
    const int      need = s_need;
    // ---- rows in order
    auto look = [&](int x, uint32_t key, bool &sure, bool &eq) {
        const bool candidate = x >= lo && x < hi;
        sure = x < r1 && (!candidate || (!none && key > top));
        eq   = x < r1 && candidate && !none && !s_done && key == top;
    };
    int n_eq = 0, n_sure = 0;
    each_row([&](int x, uint32_t key) {
        bool sure, eq;
        look(x, key, sure, eq);
        n_sure += __popc(__ballot_sync(0xffffffffu, sure));
        n_eq += __popc(__ballot_sync(0xffffffffu, eq));
    });
    // (s_eq is free: every pass ends with a barrier)
    if (lane == 0) {
        s_eq[warp]   = n_eq;
        s_sure[warp] = n_sure;
    }
    __syncthreads();
    int eq_before = (int) __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0);  // before this run
    int at = (int) __reduce_add_sync(0xffffffffu, lane < warp ? s_sure[lane] : 0) + min(eq_before, need);
    const unsigned below = (1u << lane) - 1u;
    each_row([&](int x, uint32_t key) {
        bool sure, eq;
        look(x, key, sure, eq);
        const unsigned m_eq = __ballot_sync(0xffffffffu, eq);
        const bool     stay = sure || (eq && eq_before + __popc(m_eq & below) < need);
        const unsigned m    = __ballot_sync(0xffffffffu, stay);
        if (stay) {
            const int to = at + __popc(m & below);
            out[to]      = x;
            if (wo) {
                wo[to] = w[x];
            }
        }
        eq_before += __popc(m_eq);
        at += __popc(m);
    });
}

// grid (64-row blocks of `keep`, Hkv, B); K and V of the block
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv8_move_kernel(const __grid_constant__ Kv8EvictParams P) {
    constexpr int kLanes = D / 16;  // 16 values each
    constexpr int kRows  = kMoveThreads / kLanes;
    constexpr int kPass  = kKv8Block / kRows;
    __shared__ int    s_row[kKv8Block];
    __shared__ float2 s_d[kKv8Block];  // scales of the row in K and V
    __shared__ float2 s_ratio[kKv8Block];  // of those scales to the block's new ones
    __shared__ float2 s_top[2];
    const int      blk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int      lo  = blk * kKv8Block;
    const int      n   = min(kKv8Block, P.keep - lo);  // rows of the block that are written
    const int32_t *kept = reinterpret_cast<const int32_t *>(P.kept + h * P.k_nb2 + b * P.k_nb3);
    auto           scales = [&](const Kv8Side &s) {
        return reinterpret_cast<float *>(reinterpret_cast<char *>(s.scale) + h * s.s_nb2 + b * s.s_nb3);
    };
    pdl_wait_primary();
    if (threadIdx.x < kKv8Block) {
        const int x = threadIdx.x;
        // written by the selection; a value that is no row moves nothing
        const int  row = x < n ? __ldcg(kept + lo + x) : -1;
        const bool on  = row >= 0 && row < P.c.n_max;
        float2     d   = on ? make_float2(scales(P.c.k)[row / kKv8Block], scales(P.c.v)[row / kKv8Block])
                            : make_float2(0.0f, 0.0f);
        s_row[x] = on ? row : -1;
        s_d[x]   = d;
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            d.x = max_nan(d.x, __shfl_xor_sync(0xffffffffu, d.x, off));
            d.y = max_nan(d.y, __shfl_xor_sync(0xffffffffu, d.y, off));
        }
        if ((x & 31) == 0) {
            s_top[x >> 5] = d;
        }
    }
    __syncthreads();
    const float   d_new[2] = {max_nan(s_top[0].x, s_top[1].x), max_nan(s_top[0].y, s_top[1].y)};
    const int     r0 = threadIdx.x / kLanes, e0 = 16 * (threadIdx.x % kLanes);
    const int8_t *sp[2] = {P.c.k.q + h * P.c.k.nb2 + b * P.c.k.nb3 + e0, P.c.v.q + h * P.c.v.nb2 + b * P.c.v.nb3 + e0};
    uint4         w[2][kPass];
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const int row = s_row[r0 + p * kRows];
        w[0][p] = w[1][p] = make_uint4(0u, 0u, 0u, 0u);
        if (row >= 0) {
            w[0][p] = __ldcs(reinterpret_cast<const uint4 *>(sp[0] + row * P.c.k.nb1));
            w[1][p] = __ldcs(reinterpret_cast<const uint4 *>(sp[1] + row * P.c.v.nb1));
        }
    }
    if (threadIdx.x < kKv8Block) {
        const float2 d       = s_d[threadIdx.x];
        s_ratio[threadIdx.x] = make_float2(__fdiv_rn(d.x, d_new[0]), __fdiv_rn(d.y, d_new[1]));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Kv8Side &dst = i ? P.out.v : P.out.k;
        int8_t        *dp  = dst.q + (int64_t) lo * dst.nb1 + h * dst.nb2 + b * dst.nb3 + e0;
#pragma unroll
        for (int p = 0; p < kPass; ++p) {
            const int   r = r0 + p * kRows;
            const float d = i ? s_d[r].y : s_d[r].x;
            if (d < d_new[i]) {  // (not beside a NaN scale: its block's rows keep their bytes, places without a row 0)
                const float ratio = i ? s_ratio[r].y : s_ratio[r].x;
                w[i][p].x = requant4(w[i][p].x, d, d_new[i], ratio);
                w[i][p].y = requant4(w[i][p].y, d, d_new[i], ratio);
                w[i][p].z = requant4(w[i][p].z, d, d_new[i], ratio);
                w[i][p].w = requant4(w[i][p].w, d, d_new[i], ratio);
            }
            if (r < n) {
                *reinterpret_cast<uint4 *>(dp + r * dst.nb1) = w[i][p];
            }
        }
    }
    if (threadIdx.x < 2) {
        scales(threadIdx.x ? P.out.v : P.out.k)[blk] = d_new[threadIdx.x];
    }
}

}  // namespace

cudaError_t launch_kv8_evict(const Kv8EvictParams &p, cudaStream_t s) {
    const dim3  sel((unsigned) p.c.Hkv, (unsigned) p.c.B);
    cudaError_t e;
    if (p.c.n_max <= kSelRegs * kSelThreads) {
        e = launch_pdl(kv8_select_kernel<kSelRegs>, sel, kSelThreads, 0, s, p);
    } else if (p.c.n_max <= kSelMaxKeys) {
        static thread_local int configured = -1;
        int                     dev        = 0;
        cudaGetDevice(&dev);
        if (configured != dev) {
            e = cudaFuncSetAttribute(kv8_select_kernel<kShared>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     kSelMaxKeys * (int) sizeof(uint32_t));
            if (e != cudaSuccess) {
                return e;
            }
            configured = dev;
        }
        e = launch_pdl(kv8_select_kernel<kShared>, sel, kSelThreads, (size_t) p.c.n_max * sizeof(uint32_t), s, p);
    } else {
        e = launch_pdl(kv8_select_kernel<kAgain>, sel, kSelThreads, 0, s, p);
    }
    if (e != cudaSuccess) {
        return e;
    }
    const dim3 move((unsigned) ((p.keep + kKv8Block - 1) / kKv8Block), (unsigned) p.c.Hkv, (unsigned) p.c.B);
    return p.c.D == 128 ? launch_pdl(kv8_move_kernel<128>, move, kMoveThreads, 0, s, p)
                        : launch_pdl(kv8_move_kernel<64>, move, kMoveThreads, 0, s, p);
}

}  // namespace acefa
