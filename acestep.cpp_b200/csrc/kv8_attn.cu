// kv8_attn.cu -- attention of a few query rows per KV head over the 8-bit
// block-scaled cache (acefa_kv8_attn): split over the keys, merged by a second
// launch, which also adds up the attention weights of each key.
//
// Mathematics.  With K = kd * k8 and V = vd * v8 (one kd, vd per 64 keys),
//   s_rj = scale * kd_j * (q_r . k8_j),   p_rj = exp(s_rj - m_r),
//   o_r  = sum_j vd_j p_rj v8_j / sum_j p_rj.
// k8 and v8 are integers below 128, exact in F16.  An F32 q_r (scaled by a power
// of two into F16's range) and, unless Q and the output both have 16 bits, the
// p_rj are split into two F16 numbers each, which together keep 22 bits, so that
// the F16 tensor-core products with F32 sums lose nothing beside F32 arithmetic
// (a 16-bit q_r is exact in one, and one rounding of p_rj to 11 bits is below a
// 16-bit output's own).  F16's steps end at 2^-24; m_r is therefore kept 2^kLift
// below the running maximum, and p_rj reaches from 2^15 down: what its halves
// cannot hold is below 2^-32 of the row's largest weight, so that thousands of
// keys far below one early key still count.  The scales multiply in F32: kd on
// the finished score, vd on the 16-key partial product of V.  Up to four rows,
// the two halves of a split operand ride in one product as columns r and r + 4
// of its eight.
//
// Work.  The (set, KV head, row block) units' 64-key tiles, numbered one after
// another over all sets' actual lengths, are cut into equal runs, one per CTA:
// ragged batches balance as well as even ones, and the grid depends on shapes
// only.  A unit counts as kUnitCost places more than it has tiles, about what
// beginning and merging it takes (without them a CTA could get many
// units of one tile: 8 sets of 1 .. 2560 rows took 18 us instead of 10).  A producer warp streams a CTA's tiles by TMA through a ring of stages,
// their two scales beside them by cp.async; four consumer warps take 16 keys of
// every tile each and meet only at the end of a unit.  The dims and keys of
// a fragment are assigned such that a thread's bytes are 16-B pieces of rows
// (dims are summed over in any order, and V's dims are only named at the end),
// and the boxes' layouts (K in rows of 64 B, V swizzled) such that reading the
// pieces meets no bank conflicts.
// Few short units (CL): a thread-block cluster takes each unit instead, its CTAs
// an equal share of its tiles, and the partial results meet in distributed shared
// memory -- one launch, no table of the sets, no partials in HBM.
// Measured (B200): 16 sets of up to 8192 rows, 8 KV heads, D = 128, BF16 rows:
// 47-51 us with the second launch, 4.9-5.2 TB/s in all and 6.9 TB/s between the first and
// the last tile (bound by HBM and, closely, by the four warps' instructions: 0.70 us per
// tile and CTA); 2 sets of 700 rows: 6 us, bound by the latencies of launch, Q and merge.
// Products run transposed (keys or dims are the MMA's M, the rows its N = 8):
// S^T = K Q^T and O^T = V^T P^T; P moves from the accumulator layout to the
// operand layout by four movmatrix.  m_r moves only when a score exceeds the
// maximum that it was taken from by more than 2^8 (a warp vote), as in the other kernels.
#include <algorithm>
#include <type_traits>

#include "kv8_internal.h"
#include "ptx.cuh"

namespace acefa {
namespace {

constexpr int   kWarps   = 4;  // consumers
constexpr int   kThreads = 32 * (kWarps + 1);
constexpr int   kChunk   = 16;  // keys of one warp and tile
constexpr float kSlack   = 8.0f;
constexpr float kLift    = 7.0f;  // kSlack + kLift = 15: the largest weight is 2^15, F16 holds 2^16
constexpr int   kUnitCost = 2;
// "No maximum yet": below every score, finite so that differences stay numbers
// (2^(anything - it) only meets weights and sums that are 0).
constexpr float kNoMax = -1.7e38f;
static_assert(kWarps * kChunk == kKv8Block, "a tile is one block of the cache");

// A stage: 64 rows of K (boxes of 64 dims) and of V.
template <int HD>
constexpr int stage_bytes() {
    return 2 * kKv8Block * HD;
}
template <int HD, int NT>
constexpr int stages() {
    return HD == 128 ? (NT == 2 ? 4 : 5) : 8;
}
template <int HD, int NT>
constexpr int merge_floats() {
    return kWarps * 8 * NT * (HD + 4) + kWarps * 8 * NT * 2;
}
// ring (1 KB aligned), merged rows, barriers and flag, scales of the stages, the sets' tile table and lengths
template <int HD, int NT>
constexpr int attn_smem_bytes(int B) {
    return 1024 + stages<HD, NT>() * stage_bytes<HD>() + 4 * merge_floats<HD, NT>() + (2 * stages<HD, NT>() + 1) * 8 +
           stages<HD, NT>() * 8 + 4 * (2 * B + 2);
}
constexpr int kCtasPerSm = 2;

// How operands of more than 11 bits enter the products.
constexpr int kOne    = 0;  // one F16 number (16-bit Q and output)
constexpr int kSplit  = 1;  // two, in products of their own
constexpr int kPacked = 2;  // two, as columns r and r + 4 (up to four rows)

// 4 bytes global -> shared; the barrier counts this thread as arrived when they have landed.
__device__ __forceinline__ void cp4_arrive(uint32_t dst, const void *src, uint64_t *bar) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds_v2(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
// Two bytes of `biased` (int8 + 128, picked by sel) as f16: 0x6400 | b is
// 1024 + b, and subtracting 1152 leaves the int8 value exactly.
__device__ __forceinline__ uint32_t i8x2_f16(uint32_t biased, uint32_t sel) {
    const uint32_t t = __byte_perm(biased, 0x64646464u, sel);
    const __half2  v = __hsub2(*reinterpret_cast<const __half2 *>(&t), __half2half2(__ushort_as_half(0x6480u)));
    return *reinterpret_cast<const uint32_t *>(&v);
}
// x = hi + lo as two f16 pairs, hi the rounded value
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2  f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi              = *reinterpret_cast<const uint32_t *>(&h);
    lo              = *reinterpret_cast<const uint32_t *>(&l);
}

// This thread's HD / 4 values of a Q row (zeros without one): four from dim
// 64 * (ks / 4) + 16 * c + 4 * (ks % 4) for each k-step.  The type and the
// alignment are looked at once, so that all loads leave together.
template <int HD>
__device__ __forceinline__ void load_q(const char *p, int type, int c, float (&x)[HD / 16][4]) {
    constexpr int KS = HD / 16;
    auto          at = [&](int ks) { return 64 * (ks >> 2) + 16 * c + 4 * (ks & 3); };
    if (!p) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            x[ks][0] = x[ks][1] = x[ks][2] = x[ks][3] = 0.0f;
        }
    } else if (type == ACEFA_TYPE_F32) {
        const float *f = reinterpret_cast<const float *>(p);
        if ((reinterpret_cast<uintptr_t>(f) & 15u) == 0) {
            float4 v[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                v[ks] = *reinterpret_cast<const float4 *>(f + at(ks));
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x[ks][0] = v[ks].x, x[ks][1] = v[ks].y, x[ks][2] = v[ks].z, x[ks][3] = v[ks].w;
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[ks][e] = f[at(ks) + e];
                }
            }
        }
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
        uint2           w[KS];
        if ((reinterpret_cast<uintptr_t>(h) & 7u) == 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                w[ks] = *reinterpret_cast<const uint2 *>(h + at(ks));
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint16_t *q = h + at(ks);
                w[ks] = make_uint2(q[0] | (uint32_t) q[1] << 16, q[2] | (uint32_t) q[3] << 16);
            }
        }
        const bool f16 = type == ACEFA_TYPE_F16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t v = e < 2 ? w[ks].x : w[ks].y;
                const uint32_t b = e & 1 ? v >> 16 : v & 0xFFFFu;
                x[ks][e] = f16 ? __half2float(__ushort_as_half((uint16_t) b)) : __uint_as_float(b << 16);
            }
        }
    }
}
__device__ __forceinline__ void store1(char *p, int type, int e, float x) {
    if (type == ACEFA_TYPE_F32) {
        reinterpret_cast<float *>(p)[e] = x;
    } else if (type == ACEFA_TYPE_F16) {
        reinterpret_cast<__half *>(p)[e] = __float2half_rn(x);
    } else {
        reinterpret_cast<__nv_bfloat16 *>(p)[e] = __float2bfloat16_rn(x);
    }
}

// Four finished dims of a row (L = its sum; 0: it saw nothing).
__device__ __forceinline__ void store_row4(const Kv8AttnParams &P, int row, int hk, int b, int d4, float4 o, float L) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    char *p = P.dst.data + (int64_t) (hk * P.G + row % P.G) * P.dst.nb1 + (int64_t) (row / P.G) * P.dst.nb2 +
              (int64_t) b * P.dst.nb3;
    store1(p, P.dst.type, 4 * d4, o.x * inv);
    store1(p, P.dst.type, 4 * d4 + 1, o.y * inv);
    store1(p, P.dst.type, 4 * d4 + 2, o.z * inv);
    store1(p, P.dst.type, 4 * d4 + 3, o.w * inv);
}

// base[b] = places of one unit of each set before b, b = 0 .. B: its 64-key tiles
// and, ahead of them, kUnitCost (none without tiles); lens[b] = length.  All
// threads; ends with a barrier.
__device__ __forceinline__ void tile_table(int *base, int *lens, const int32_t *len, int B, int n_max) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
        int acc = 0;
        for (int b0 = 0; b0 < B; b0 += 32) {
            const int n = b0 + lane < B ? clamp_len(len[b0 + lane], n_max) : 0;
            int       v = n ? (n + kKv8Block - 1) / kKv8Block + kUnitCost : 0;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, off);
                v += lane >= off ? u : 0;
            }
            if (b0 + lane < B) {
                base[b0 + lane + 1] = acc + v;
                lens[b0 + lane]     = n;
            }
            acc += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) {
            base[0] = 0;
        }
    }
    __syncthreads();
}

// Run of places of CTA c of C: [T * c / C, T * (c + 1) / C).  C <= T, so no run
// is empty and the CTAs that meet a unit's tiles are consecutive.
__device__ __forceinline__ int run_start(int T, int C, int c) { return (int) ((int64_t) T * c / C); }
// the CTA whose run holds place x
__device__ __forceinline__ int cta_of(int T, int C, int x) { return (int) ((((int64_t) x + 1) * C - 1) / T); }

// A position in the sequence of tiles.
struct Walk {
    int b, ub, t, nt, len;  // set, unit of the set, tile of the unit, its tiles, the set's length
    int at;                 // place
};

// D = A B (a product that starts a sum)
__device__ __forceinline__ void mma_start(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <int HD, int NT, int MODE, bool CL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    kv8_attn_kernel(const __grid_constant__ Kv8AttnParams P, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap) {
    constexpr int R       = 8 * NT;
    constexpr int KS      = HD / 16;  // k-steps of S, m-tiles of O
    constexpr int kSt     = stage_bytes<HD>();
    constexpr int kStages = stages<HD, NT>();
    constexpr int kOut    = HD + 4;  // floats between merged rows
    extern __shared__ uint8_t smem_raw[];
    uint8_t  *smem   = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float    *s_o    = reinterpret_cast<float *>(smem + kStages * kSt);  // [warp][R][kOut]
    float    *s_ml   = s_o + kWarps * R * kOut;                          // [warp][R][2]
    uint64_t *full   = reinterpret_cast<uint64_t *>(s_ml + kWarps * R * 2);
    uint64_t *empty  = full + kStages;
    volatile int *abort_f = reinterpret_cast<volatile int *>(empty + kStages);
    float    *s_sc   = reinterpret_cast<float *>(empty + kStages + 1);  // [stage][K, V]
    int      *s_base = reinterpret_cast<int *>(s_sc + 2 * kStages);
    int      *s_len  = s_base + P.c.B + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    const int HU = P.c.Hkv * P.n_rb;  // units of a set

    if (threadIdx.x == kThreads - 1) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 3);  // the boxes, and a scale each
            mbar_init(&empty[i], kWarps);
        }
        *abort_f = 0;
        fence_barrier_init();
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
    }
    pdl_wait_primary();
    Walk at;
    int  x1;  // behind the last place of this CTA's run
    if constexpr (CL) {
        const int unit = (int) blockIdx.x / P.cluster, rank = (int) blockIdx.x - unit * P.cluster;
        at.b   = unit / HU;
        at.ub  = unit - at.b * HU;
        at.len = clamp_len(P.len[at.b], P.c.n_max);
        at.nt  = (at.len + kKv8Block - 1) / kKv8Block;
        at.t = at.at = run_start(at.nt, P.cluster, rank);
        x1           = run_start(at.nt, P.cluster, rank + 1);
        __syncthreads();
    } else {
        tile_table(s_base, s_len, P.len, P.c.B, P.c.n_max);
        const int T = s_base[P.c.B] * HU;
        const int C = min((int) gridDim.x, T);
        // The sum kernel, always the next in the stream, may be set up from here on.  It reads the
        // lengths before its own wait, which is sound only behind this one's pdl_wait_primary():
        // whatever wrote them is complete.
        pdl_launch_dependents();
        if ((int) blockIdx.x >= C) {
            return;
        }
        const int x0 = run_start(T, C, blockIdx.x);
        x1           = run_start(T, C, blockIdx.x + 1);
        // the set whose places hold x0: base[b] * HU <= x0 < base[b + 1] * HU, by 32nds
        int lo = 0, n = P.c.B;
        while (n > 1) {
            const int step = (n + 31) >> 5, i = lo + lane * step;
            const int below = __popc(__ballot_sync(0xffffffffu, lane * step < n && s_base[i] * HU <= x0));
            n  = min(step, n - (below - 1) * step);
            lo += (below - 1) * step;
        }
        at.b          = lo;
        const int per = s_base[lo + 1] - s_base[lo];
        at.nt         = per - kUnitCost;
        at.len        = s_len[lo];
        const int off = x0 - s_base[lo] * HU;
        at.ub         = (int) ((unsigned) off / (unsigned) per);
        const int r   = off - at.ub * per;
        at.t          = max(r - kUnitCost, 0);
        at.at         = x0 + max(kUnitCost - r, 0);
        if (at.at >= x1) {
            return;  // no tile in this run
        }
    }

    auto advance = [&](Walk &w) {  // true: a new unit
        ++w.at;
        if (++w.t < w.nt || CL) {
            return false;
        }
        w.t = 0;
        w.at += kUnitCost;
        if (++w.ub == HU) {
            w.ub = 0;
            do {
                ++w.b;
            } while (w.b < P.c.B && s_base[w.b + 1] == s_base[w.b]);
            if (w.b == P.c.B) {
                return true;
            }
            w.nt  = s_base[w.b + 1] - s_base[w.b] - kUnitCost;
            w.len = s_len[w.b];
        }
        return true;
    };
    auto kv_head = [&](const Walk &w) { return P.n_rb == 1 ? w.ub : w.ub / P.n_rb; };
    // This thread's row of Q of a unit (kPacked: rows 4 .. 7 are the low halves of 0 .. 3), or nullptr
    auto q_row = [&](const Walk &w, int nt, int &row) -> const char * {
        const int hk = kv_head(w);
        row          = (w.ub - hk * P.n_rb) * R + nt * 8 + (MODE == kPacked ? g & 3 : g);
        const int iq = P.n_q == 1 ? 0 : row / P.G;
        return row < P.rows ? P.q.data + iq * P.q.nb1 + (int64_t) (hk * P.G + row - iq * P.G) * P.q.nb2 +
                                  (int64_t) w.b * P.q.nb3
                            : nullptr;
    };

    if (warp == kWarps) {
        // ============================ producer =================================
        const float *ksp = nullptr, *vsp = nullptr;  // the tile's scales
        int          hk = 0;
        auto         aim = [&]() {
            hk  = kv_head(at);
            ksp = reinterpret_cast<const float *>(reinterpret_cast<const char *>(P.c.k.scale) + hk * P.c.k.s_nb2 +
                                                  at.b * P.c.k.s_nb3) +
                  at.t;
            vsp = reinterpret_cast<const float *>(reinterpret_cast<const char *>(P.c.v.scale) + hk * P.c.v.s_nb2 +
                                                  at.b * P.c.v.s_nb3) +
                  at.t;
        };
        aim();
        bool     ok = true;
        int      st = 0;
        uint32_t ph = 0;
        while (at.at < x1) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], ph ^ 1u, abort_f, P.dev_err, DEVERR_TIMEOUT_EMPTY,
                                                           P.wait_limit_ns));
            if (!ok) {
                break;
            }
            if (lane == 0) {
                uint8_t *dst = smem + st * kSt;
                mbar_arrive_expect_tx(&full[st], kSt);
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) {
                    tma_load_4d(dst + e * (kKv8Block * 64), &kmap, 64 * e, at.t * kKv8Block, hk, at.b, &full[st]);
                }
                tma_load_4d(dst + kKv8Block * HD, &vmap, 0, at.t * kKv8Block, hk, at.b, &full[st]);
            } else if (lane == 1) {
                cp4_arrive(smem_u32(s_sc + 2 * st), ksp, &full[st]);
            } else if (lane == 2) {
                cp4_arrive(smem_u32(s_sc + 2 * st + 1), vsp, &full[st]);
            }
            if (++st == kStages) {
                st = 0;
                ph ^= 1u;
            }
            if (!advance(at)) {
                ++ksp, ++vsp;
            } else if (!CL && at.b < P.c.B) {
                aim();
                if (at.at < x1) {  // the next unit's rows of Q, on their way to L1
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        int         row;
                        const char *p = q_row(at, nt, row);
                        if (p) {
                            asm volatile("prefetch.global.L1 [%0];" ::"l"(p + (P.q.type == ACEFA_TYPE_F32 ? HD : HD / 2) * c));
                        }
                    }
                }
            }
            __syncwarp();
        }
        if (!ok) {
            // let the copies in flight land before the CTA exits
            const uint64_t ts = globaltimer_ns();
            for (int i = 0; i < kStages; ++i) {
                const uint32_t last = i < st ? ph : ph ^ 1u;  // the last use of stage i, if it had one
                while (!mbar_try_wait(&full[i], last)) {
                    if (globaltimer_ns() - ts > P.wait_limit_ns) {
                        break;
                    }
                }
            }
        }
        return;
    }

    // ---- rows of the current unit
    uint32_t qh[NT][KS][2], ql[MODE == kSplit ? NT : 1][KS][2];  // Q^T operand, its (other) half
    float    mul[NT][2];                    // log2-unit score per unit of accumulator, rows 2c and 2c + 1
    int      lim[NT][2];                    // keys those rows see
    float    acc_o[NT][KS][4];
    float    m[NT][2], l[NT][2];
    float   *sp = nullptr;  // this thread's scores of the chunk, where weights are wanted
    auto start_rows = [&]() {
        const int rb = at.ub - kv_head(at) * P.n_rb;
        if (P.scores) {
            sp = P.scores + ((int64_t) (at.b * HU + at.ub) * P.c.n_max + at.t * kKv8Block + warp * kChunk + g) * P.score_stride +
                 2 * c;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            int         row;
            const char *p = q_row(at, nt, row);
            float       x[KS][4], top = 0.0f;
            load_q<HD>(p, P.q.type, c, x);  // (the dims of the words of this thread's K pieces)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = fmaxf(top, fabsf(x[ks][e]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^k brings the row's largest value into [2^13, 2^14): far below
            // F16's largest, and small values keep their bits in the low half
            const int ex = (int) (__float_as_uint(top) >> 23);
            const int k  = top > 0.0f && ex < 255 ? min(140 - ex, 126) : 0;
            const float f = __uint_as_float((uint32_t) (127 + k) << 23);
            const float u = P.scale_log2 * __uint_as_float((uint32_t) (127 - k) << 23);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t hi, lo;
                    split2(x[ks][2 * e] * f, x[ks][2 * e + 1] * f, hi, lo);
                    qh[nt][ks][e] = MODE == kPacked && g >= 4 ? lo : hi;
                    if constexpr (MODE == kSplit) {
                        ql[nt][ks][e] = lo;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mul[nt][e]    = __shfl_sync(0xffffffffu, u, (2 * c + e) * 4);
                const int rr  = rb * R + nt * 8 + (MODE == kPacked ? (2 * c + e) & 3 : 2 * c + e);
                const int iq  = P.n_q == 1 ? 0 : rr / P.G;
                lim[nt][e]    = rr < P.rows ? at.len - (P.n_q - 1 - iq) : 0;
                m[nt][e]      = kNoMax;
                l[nt][e]      = 0.0f;
            }
#pragma unroll
            for (int t = 0; t < KS; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc_o[nt][t][e] = 0.0f;
                }
            }
        }
    };

    // The four warps' results of a unit as one: n_row rows of HD at dst, R maxima
    // and R sums behind R rows.
    auto merge = [&](float *dst, int n_row) {
        named_bar_sync(1, 32 * kWarps);  // the previous merge has been read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[nt][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = nt * 8 + 2 * c + e;
                if (g == 0) {
                    s_ml[(warp * R + row) * 2]     = m[nt][e];
                    s_ml[(warp * R + row) * 2 + 1] = sum;
                }
                // element e of the accumulators is dim 2t of row 2c + e, element 2 + e dim 2t + 1
                float *o = s_o + (warp * R + row) * kOut + g * (HD / 8);
#pragma unroll
                for (int t = 0; t < KS; t += 2) {
                    *reinterpret_cast<float4 *>(o + 2 * t) = make_float4(acc_o[nt][t][e], acc_o[nt][t][2 + e],
                                                                         acc_o[nt][t + 1][e], acc_o[nt][t + 1][2 + e]);
                }
            }
        }
        named_bar_sync(1, 32 * kWarps);
        if (MODE == kPacked) {
            n_row = min(n_row, 4);
        }
        for (int x = threadIdx.x; x < n_row * (HD / 4); x += 32 * kWarps) {
            const int row = x / (HD / 4), d4 = x % (HD / 4);
            float     mw[kWarps], M = kNoMax;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                mw[w] = s_ml[(w * R + row) * 2];
                M     = fmaxf(M, mw[w]);
            }
            float  L = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2f(mw[w] - M);
                float4      v = *reinterpret_cast<const float4 *>(s_o + (w * R + row) * kOut + 4 * d4);
                if constexpr (MODE == kPacked) {
                    const float4 u = *reinterpret_cast<const float4 *>(s_o + (w * R + row + 4) * kOut + 4 * d4);
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                }
                L += s_ml[(w * R + row) * 2 + 1] * f;
                o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
            }
            *reinterpret_cast<float4 *>(dst + row * HD + 4 * d4) = o;
            if (d4 == 0) {
                dst[R * HD + row]     = M;
                dst[R * HD + R + row] = L;
            }
        }
    };
    start_rows();
    // K row g of this warp's chunk, 16-B piece c; V rows 2c .. of it, HD / 8 dims of g
    const uint32_t k_at = smem_u32(smem) + (uint32_t) ((warp * kChunk + g) * 64 + 16 * c);
    const uint32_t v_at = smem_u32(smem) + (uint32_t) (kKv8Block * HD + (warp * kChunk + 2 * c) * HD);
    int            stage = 0;
    uint32_t       phase = 0;
    bool           ok    = true;

#pragma unroll 1
    while (at.at < x1) {
        const int j0 = at.t * kKv8Block + warp * kChunk;
        // (after an expired wait the loop runs on without data, to meet the others at the barriers)
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], phase, abort_f, P.dev_err, DEVERR_TIMEOUT_FULL,
                                                       P.wait_limit_ns)) && ok;
        if (ok && j0 < at.len) {  // uniform over the warp
            const float kd = s_sc[2 * stage];
            float       vd = s_sc[2 * stage + 1];
            // ---- S^T = K Q^T
            // (two sums per product, of the even and the odd k-steps: half as long a chain)
            float s[NT][4], s2[NT][MODE == kSplit ? 3 : 1][4];
#pragma unroll
            for (int e4 = 0; e4 < HD / 64; ++e4) {
                const uint32_t ka    = k_at + (uint32_t) (stage * kSt + e4 * (kKv8Block * 64));
                const uint4    wa    = lds_v4(ka);
                const uint4    wb    = lds_v4(ka + 8 * 64);
                const uint32_t va[4] = {wa.x, wa.y, wa.z, wa.w}, vb[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t ba = va[e] ^ 0x80808080u, bb = vb[e] ^ 0x80808080u;
                    const uint32_t a[4] = {i8x2_f16(ba, 0x4140u), i8x2_f16(bb, 0x4140u), i8x2_f16(ba, 0x4342u),
                                           i8x2_f16(bb, 0x4342u)};
                    const int      ks   = 4 * e4 + e;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float(&sum)[4] = e & 1 ? s2[nt][0] : s[nt];
                        if (ks < 2) {
                            mma_start(sum, a, qh[nt][ks][0], qh[nt][ks][1]);
                        } else {
                            mma_16816<false>(sum, a, qh[nt][ks][0], qh[nt][ks][1]);
                        }
                        if constexpr (MODE == kSplit) {
                            if (ks < 2) {
                                mma_start(s2[nt][1 + (e & 1)], a, ql[nt][ks][0], ql[nt][ks][1]);
                            } else {
                                mma_16816<false>(s2[nt][1 + (e & 1)], a, ql[nt][ks][0], ql[nt][ks][1]);
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nt][e] += s2[nt][0][e];
                    if constexpr (MODE == kSplit) {
                        s[nt][e] += s2[nt][1][e] + s2[nt][2][e];
                    }
                    if constexpr (MODE == kPacked) {  // columns r and r + 4
                        s[nt][e] += __shfl_xor_sync(0xffffffffu, s[nt][e], 2);
                    }
                }
            }
            // ---- scores in log2 units, masked; s[nt]: (key g, rows 2c 2c+1), (key g + 8, same rows)
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float u = mul[nt][e] * kd;
                    s[nt][e] *= u;
                    s[nt][2 + e] *= u;
                }
            }
            if (j0 + kChunk > at.len - (P.n_q - 1)) {  // keys that some row does not see
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[nt][e] = j0 + g + 8 * (e >> 1) < lim[nt][e & 1] ? s[nt][e] : -INFINITY;
                    }
                }
                if (!(fabsf(vd) < INFINITY)) {
                    // V's scale is no number, and 0 * NaN would reach the rows that see
                    // nothing of the chunk: the others' sums become NaN here
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
#pragma unroll
                            for (int t = 0; t < KS; ++t) {
                                acc_o[nt][t][e] = j0 < lim[nt][e & 1] ? NAN : acc_o[nt][t][e];
                            }
                        }
                    }
                    vd = 0.0f;
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    grow |= fmaxf(s[nt][e], s[nt][2 + e]) > m[nt][e] + (kSlack + kLift);
                }
            }
            if (P.scores) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (nt * 8 + 2 * c < P.score_stride && j0 + g + 8 * e < at.len) {
                            *reinterpret_cast<float2 *>(sp + 8 * e * P.score_stride + nt * 8) =
                                make_float2(s[nt][2 * e], s[nt][2 * e + 1]);
                        }
                    }
                }
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(s[nt][e], s[nt][2 + e]);
                        top       = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top       = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top       = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float mn = fmaxf(m[nt][e], top - kLift);
                        const float f  = fast_exp2(m[nt][e] - mn);
                        m[nt][e]       = mn;
                        l[nt][e] *= f;
#pragma unroll
                        for (int t = 0; t < KS; ++t) {
                            acc_o[nt][t][e] *= f;
                            acc_o[nt][t][2 + e] *= f;
                        }
                    }
                }
            }
            // ---- P, its operand halves
            uint32_t ph[NT][2], pl[MODE == kSplit ? NT : 1][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = fast_exp2(s[nt][e] - m[nt][e & 1]);
                    l[nt][e & 1] += p[e];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t hi, lo;
                    split2(p[2 * e], p[2 * e + 1], hi, lo);
                    ph[nt][e] = movmatrix_trans(MODE == kPacked && c >= 2 ? lo : hi);
                    if constexpr (MODE == kSplit) {
                        pl[nt][e] = movmatrix_trans(lo);
                    }
                }
            }
            // ---- O^T += vd * V^T P^T.  m-tile t: dims g * HD / 8 + 2t (row g) and + 2t + 1 (row g + 8)
            uint32_t v[4][HD / 32];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int      row = (r & 1) + 8 * (r >> 1);  // from 2c
                const uint32_t va  = v_at + (uint32_t) (stage * kSt + row * HD);
                if constexpr (HD == 128) {  // 128-B swizzle: piece ^ (row & 7)
                    const uint4 w = lds_v4(va + (uint32_t) ((g ^ (2 * c + (r & 1))) << 4));
                    v[r][0] = w.x, v[r][1] = w.y, v[r][2] = w.z, v[r][3] = w.w;
                } else {  // 64-B swizzle: piece ^ ((row >> 1) & 3)
                    const uint2 w = lds_v2(va + (uint32_t) (((g >> 1) ^ c) << 4) + 8 * (g & 1));
                    v[r][0] = w.x, v[r][1] = w.y;
                }
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&empty[stage]);  // the warp's bytes are in registers
            }
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                const uint32_t sel = (t & 1) ? 0x7362u : 0x5140u;
                const uint32_t z0  = __byte_perm(v[0][t >> 1], v[1][t >> 1], sel) ^ 0x80808080u;
                const uint32_t z1  = __byte_perm(v[2][t >> 1], v[3][t >> 1], sel) ^ 0x80808080u;
                const uint32_t a[4] = {i8x2_f16(z0, 0x4140u), i8x2_f16(z0, 0x4342u), i8x2_f16(z1, 0x4140u),
                                       i8x2_f16(z1, 0x4342u)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float o[4];
                    mma_start(o, a, ph[nt][0], ph[nt][1]);
                    if constexpr (MODE == kSplit) {
                        mma_16816<false>(o, a, pl[nt][0], pl[nt][1]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc_o[nt][t][e] = fmaf(o[e], vd, acc_o[nt][t][e]);
                    }
                }
            }
        }
        else if (lane == 0) {
            mbar_arrive(&empty[stage]);
        }
        // ---- end of the unit (or of this CTA's run): merge the warps' results
        const int  unit = at.b * HU + at.ub;
        const int  rb   = at.ub - kv_head(at) * P.n_rb;
        const bool next = advance(at);
        if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
        }
        if (P.scores) {
            sp += kKv8Block * P.score_stride;
        }
        if (!CL && (next || at.at >= x1)) {
            merge(P.part + (int64_t) (blockIdx.x + unit) * (R * (HD + 2)), min(R, P.rows - rb * R));
            if (at.at < x1) {
                start_rows();
            }
        }
    }
    if constexpr (CL) {
        // Every CTA's result to its own shared memory (the ring is empty: each of
        // its tiles has been awaited), then the cluster's CTAs finish a share of
        // the unit's values each from all of them.
        float *fin = reinterpret_cast<float *>(smem);
        merge(fin, R);
        cluster_arrive();
        cluster_wait();
        const int      rank = (int) cluster_ctarank(), hk = kv_head(at), rb = at.ub - hk * P.n_rb;
        const int      n_row = min(R, P.rows - rb * R);
        const uint32_t f_at  = smem_u32(fin);
        for (int x = (int) threadIdx.x * P.cluster + rank; x < n_row * (HD / 4); x += 32 * kWarps * P.cluster) {
            const int r = x / (HD / 4), d4 = x % (HD / 4);
            float     m8[8], l8[8], M = kNoMax, L = 0.0f;
            float4    o8[8], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // every value asked for at once
                if (k < P.cluster) {
                    const uint32_t p = mapa_shared(f_at, (uint32_t) k);
                    m8[k] = ld_cluster_f32(p + 4u * (R * HD + r));
                    l8[k] = ld_cluster_f32(p + 4u * (R * HD + R + r));
                    o8[k] = ld_cluster_f32x4(p + 4u * (r * HD + 4 * d4));
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                M = k < P.cluster ? fmaxf(M, m8[k]) : M;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k < P.cluster) {
                    const float f = exp2f(m8[k] - M);
                    L = fmaf(l8[k], f, L);
                    o.x = fmaf(o8[k].x, f, o.x), o.y = fmaf(o8[k].y, f, o.y);
                    o.z = fmaf(o8[k].z, f, o.z), o.w = fmaf(o8[k].w, f, o.w);
                }
            }
            store_row4(P, rb * R + r, hk, at.b, d4, o, L);
        }
        if (P.weight) {  // (n_rb == 1) this CTA's own keys
            float *s_lse = s_ml;  // free: the merge is behind the cluster's barrier
            for (int r = threadIdx.x; r < n_row; r += 32 * kWarps) {
                float M = kNoMax, L = 0.0f;
                for (int k = 0; k < P.cluster; ++k) {
                    M = fmaxf(M, ld_cluster_f32(mapa_shared(f_at, (uint32_t) k) + 4u * (R * HD + r)));
                }
                for (int k = 0; k < P.cluster; ++k) {
                    const uint32_t q = mapa_shared(f_at, (uint32_t) k) + 4u * (R * HD + r);
                    L = fmaf(ld_cluster_f32(q + 4u * R), exp2f(ld_cluster_f32(q) - M), L);
                }
                s_lse[r] = L == 0.0f ? INFINITY : M + log2f(L);  // an empty row weighs nothing
            }
            cluster_arrive_relaxed();  // the peers' memory is read
            named_bar_sync(1, 32 * kWarps);  // (and orders the scores that the warps of this CTA wrote)
            const int j0 = run_start(at.nt, P.cluster, rank) * kKv8Block, j1 = min(at.len, x1 * kKv8Block);
            float    *wp = reinterpret_cast<float *>(P.weight + (int64_t) hk * P.w_nb2 + (int64_t) at.b * P.w_nb3);
            const float2 *sc = reinterpret_cast<const float2 *>(P.scores + (int64_t) (at.b * HU + at.ub) * P.c.n_max * P.score_stride);
            constexpr int kAtOnce = R == 8 ? 4 : 2;  // keys of a thread on their way together
            for (int jb = j0 + (int) threadIdx.x; jb < j1; jb += kAtOnce * 32 * kWarps) {
                float2 v[kAtOnce][R / 2];
                float  w[kAtOnce], sum[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const int j = jb + k * 32 * kWarps;
                    w[k]        = j < j1 ? wp[j] : 0.0f;
                    sum[k]      = 0.0f;
#pragma unroll
                    for (int r = 0; r < R / 2; ++r) {
                        v[k][r] = j < j1 && 2 * r < P.score_stride ? __ldcg(sc + (int64_t) j * (P.score_stride >> 1) + r)
                                                                   : make_float2(-INFINITY, -INFINITY);
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < n_row) {
#pragma unroll
                        for (int k = 0; k < kAtOnce; ++k) {
                            sum[k] += fast_exp2((r & 1 ? v[k][r >> 1].y : v[k][r >> 1].x) - s_lse[r]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const int j = jb + k * 32 * kWarps;
                    if (j < j1) {
                        wp[j] = w[k] + sum[k];
                    }
                }
            }
        } else {
            cluster_arrive_relaxed();
        }
        cluster_wait();  // no CTA leaves while a peer reads its memory
    }
}

// ---------------------------------------------------------------------------
// The second launch.  CTAs below n_out finish one row each: O = sum of the
// partials, each times 2^(m - M), over their summed l.  The others add the
// weights of a few hundred keys of a (set, KV head): p = 2^(s - M) / L summed over the
// head's rows, whose M and L come from the same partials.  Every sum has a
// fixed order, so results do not depend on scheduling.
constexpr int kSumThreads = 128;
constexpr int kSumKeys    = 2 * kSumThreads;  // at a time
constexpr int kSumCtas    = 1024;             // about what the device holds

// A maximum and the sum of l * 2^(m - maximum), joined with another pair.
__device__ __forceinline__ void join(float &M, float &L, float m, float l) {
    const float mn = fmaxf(M, m), mu = mn == -INFINITY ? 0.0f : mn;
    L = L * fast_exp2(M - mu) + l * fast_exp2(m - mu);
    M = mn;
}
// The pairs of a row in slots c0 + first, c0 + first + step .. c1 (base: its
// first m; l is R further), four loads of each on their way at a time.
__device__ __forceinline__ void join_slots(const float *base, int64_t slot_f, int R, int first, int step, int c0, int c1,
                                           float &M, float &L) {
    M = -INFINITY;
    L = 0.0f;
    for (int k = c0 + first; k <= c1; k += 4 * step) {
        float m[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool on = k + e * step <= c1;
            m[e] = on ? __ldcg(base + (k + e * step) * slot_f) : -INFINITY;
            l[e] = on ? __ldcg(base + (k + e * step) * slot_f + R) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            join(M, L, m[e], l[e]);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kSumThreads) kv8_attn_sum_kernel(const __grid_constant__ Kv8AttnParams P, int R,
                                                                   int n_out, int key_chunks, int keys) {
    extern __shared__ __align__(16) int s_tab[];  // tile table and lengths
    __shared__ float  s_lse[ACEFA_KV8_MAX_ROWS];
    __shared__ float4 s_o[4][HD / 4];
    __shared__ float2 s_join[kSumThreads];
    int          *s_base = s_tab, *s_len = s_tab + P.c.B + 1;
    const int     lane = threadIdx.x & 31;
    const int64_t slot_f = (int64_t) R * (HD + 2);
    const int     HU     = P.c.Hkv * P.n_rb;
    // (the lengths are older than the split kernel, which let this one start only after its own wait)
    tile_table(s_base, s_len, P.len, P.c.B, P.c.n_max);
    const int T = s_base[P.c.B] * HU, C = min(P.n_cta, T);
    // the CTAs of the split kernel that met a unit: slots (c + unit), c0 <= c <= c1
    auto range_of = [&](int b, int ub, int &c0, int &c1) {
        const int per = s_base[b + 1] - s_base[b];
        const int a   = s_base[b] * HU + ub * per;
        c0 = per ? cta_of(T, C, a + kUnitCost) : 0;
        c1 = per ? cta_of(T, C, a + per - 1) : -1;
    };
    if ((int) blockIdx.x < n_out) {
        const int row = blockIdx.x % P.rows, bh = blockIdx.x / P.rows;
        const int hk = bh % P.c.Hkv, b = bh / P.c.Hkv;
        const int ub = hk * P.n_rb + row / R, r = row % R;
        int       c0, c1;
        range_of(b, ub, c0, c1);
        const float *base = P.part + (int64_t) (b * HU + ub) * slot_f;
        pdl_wait_primary();
        float M, L;
        join_slots(base + R * HD + r, slot_f, R, lane, 32, c0, c1, M, L);
#pragma unroll
        for (int off = 16; off; off >>= 1) {
            join(M, L, __shfl_xor_sync(0xffffffffu, M, off), __shfl_xor_sync(0xffffffffu, L, off));
        }
        L = __shfl_sync(0xffffffffu, L, 0);  // (the lanes' sums differ in the order of their terms)
        const float Mu = M == -INFINITY ? 0.0f : M;
        const int   w = threadIdx.x / (HD / 4), d4 = threadIdx.x % (HD / 4);
        constexpr int W = kSumThreads / (HD / 4);  // slots summed side by side
        float4      o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = c0 + w; k <= c1; k += W) {
            const float *sl = base + (int64_t) k * slot_f;
            const float  f  = exp2f(__ldcg(sl + R * HD + r) - Mu);
            const float4 v  = __ldcg(reinterpret_cast<const float4 *>(sl + r * HD) + d4);
            o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
        }
        for (int half = W / 2; half; half >>= 1) {
            if (w >= half && w < 2 * half) {
                s_o[w - half][d4] = o;
            }
            __syncthreads();
            if (w < half) {
                const float4 v = s_o[w][d4];
                o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
            }
            __syncthreads();
        }
        if (w == 0) {
            store_row4(P, row, hk, b, d4, o, L);
        }
        return;
    }
    const int x = (int) blockIdx.x - n_out;
    const int bh = x / key_chunks, j0 = x % key_chunks * keys;
    const int hk = bh % P.c.Hkv, b = bh / P.c.Hkv;
    const int len = s_len[b];
    if (j0 >= len) {
        return;
    }
    pdl_wait_primary();
    // two keys per thread; the scores of the first row block are on their way
    // while the rows' sums are put together
    const int     st    = P.score_stride;  // even
    const int     j_end = min(len, j0 + keys);
    int           j[2]  = {j0 + (int) threadIdx.x, j0 + (int) threadIdx.x + kSumThreads};
    const float2 *sp    = reinterpret_cast<const float2 *>(P.scores + (int64_t) (b * HU + hk * P.n_rb) * P.c.n_max * st);
    float2        s[2][8];
    auto          fetch = [&](int rb) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                s[k][r] = j[k] < j_end && 2 * r < st
                                       ? __ldcg(sp + ((int64_t) rb * P.c.n_max + j[k]) * (st >> 1) + r)
                                       : make_float2(-INFINITY, -INFINITY);
            }
        }
    };
    fetch(0);
    // every row's maximum and sum: thread = (row of the block, share of its slots)
    const int n_sh = kSumThreads / R, row = (int) threadIdx.x % R, sh = (int) threadIdx.x / R;
    for (int rb = 0; rb < P.n_rb; ++rb) {
        const int ub = hk * P.n_rb + rb;
        int       c0, c1;
        range_of(b, ub, c0, c1);
        float M = -INFINITY, L = 0.0f;
        if (rb * R + row < P.rows) {
            join_slots(P.part + (int64_t) (b * HU + ub) * slot_f + R * HD + row, slot_f, R, sh, n_sh, c0, c1, M, L);
        }
        s_join[threadIdx.x] = make_float2(M, L);
        __syncthreads();
        if (sh == 0 && rb * R + row < P.rows) {
            for (int k = 1; k < n_sh; ++k) {
                const float2 v = s_join[k * R + row];
                join(M, L, v.x, v.y);
            }
            // an empty row weighs nothing
            s_lse[rb * R + row] = L == 0.0f ? INFINITY : (M == -INFINITY ? 0.0f : M) + log2f(L);
        }
        __syncthreads();
    }
    float *wp = reinterpret_cast<float *>(P.weight + (int64_t) hk * P.w_nb2 + (int64_t) b * P.w_nb3);
    for (int jb = j0; jb < j_end; jb += kSumKeys) {
        float sum[2] = {0.0f, 0.0f};
        for (int rb = 0; rb < P.n_rb; ++rb) {
            if (rb) {
                fetch(rb);
            }
            const int n_row = min(R, P.rows - rb * R);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (r < n_row) {
                    const float lse = s_lse[rb * R + r];
                    sum[0] += fast_exp2((r & 1 ? s[0][r >> 1].y : s[0][r >> 1].x) - lse);
                    sum[1] += fast_exp2((r & 1 ? s[1][r >> 1].y : s[1][r >> 1].x) - lse);
                }
            }
        }
        const int w[2] = {j[0], j[1]};
        j[0] += kSumKeys, j[1] += kSumKeys;
        fetch(0);  // (nothing behind the last)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (w[k] < j_end) {
                wp[w[k]] += sum[k];
            }
        }
    }
}

// K or V of the cache as [D, n_max, Hkv, B] bytes; boxes of `inner` dims x 64 rows.
bool encode_side(CUtensorMap *map, const Kv8Dev &c, const Kv8Side &side, int inner, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) {
        return false;
    }
    // strides of extent-1 dims do not matter; keep them 16-B multiples
    const cuuint64_t s1 = c.n_max > 1 ? (cuuint64_t) side.nb1 : (cuuint64_t) c.D;
    const cuuint64_t s2 = c.Hkv > 1 ? (cuuint64_t) side.nb2 : s1 * (cuuint64_t) c.n_max;
    const cuuint64_t s3 = c.B > 1 ? (cuuint64_t) side.nb3 : s2 * (cuuint64_t) c.Hkv;
    cuuint64_t dims[4] = {(cuuint64_t) c.D, (cuuint64_t) c.n_max, (cuuint64_t) c.Hkv, (cuuint64_t) c.B};
    cuuint64_t strides[3] = {s1, s2, s3};
    cuuint32_t box[4] = {(cuuint32_t) inner, kKv8Block, 1, 1}, estr[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, side.q, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int NT, int MODE, bool CL>
cudaError_t configure(int *smem, int B) {
    *smem = attn_smem_bytes<HD, NT>(CL ? 0 : B);
    static thread_local int configured = -1;
    int                     dev        = 0;
    cudaGetDevice(&dev);
    if (configured != dev) {
        cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<HD, NT, MODE, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             attn_smem_bytes<HD, NT>(kKv8MaxSets));
        if (e != cudaSuccess) {
            return e;
        }
        configured = dev;
    }
    return cudaSuccess;
}

template <int HD, int NT, int MODE>
cudaError_t launch(const Kv8AttnParams &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t s) {
    cudaLaunchAttribute attr[2];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id                                         = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x                           = (unsigned) p.cluster;
    attr[1].val.clusterDim.y                           = 1;
    attr[1].val.clusterDim.z                           = 1;
    int                smem = 0;
    cudaLaunchConfig_t cfg  = {};
    cfg.blockDim            = dim3(kThreads);
    cfg.stream              = s;
    cfg.attrs               = attr;
    if (p.cluster) {
        cudaError_t e = configure<HD, NT, MODE, true>(&smem, p.c.B);
        if (e != cudaSuccess) {
            return e;
        }
        cfg.gridDim          = dim3((unsigned) (p.c.B * p.c.Hkv * p.n_rb * p.cluster));
        cfg.dynamicSmemBytes = (size_t) smem;
        cfg.numAttrs         = 2;
        return cudaLaunchKernelEx(&cfg, kv8_attn_kernel<HD, NT, MODE, true>, p, km, vm);
    }
    cudaError_t e = configure<HD, NT, MODE, false>(&smem, p.c.B);
    if (e != cudaSuccess) {
        return e;
    }
    cfg.gridDim          = dim3((unsigned) p.n_cta);
    cfg.dynamicSmemBytes = (size_t) smem;
    cfg.numAttrs         = 1;
    e                    = cudaLaunchKernelEx(&cfg, kv8_attn_kernel<HD, NT, MODE, false>, p, km, vm);
    if (e != cudaSuccess) {
        return e;
    }
    const int n_out = p.c.B * p.c.Hkv * p.rows;
    // keys of a CTA: enough for about kSumCtas of them in all
    const int64_t all  = (int64_t) p.c.B * p.c.Hkv * p.c.n_max;
    const int     keys = (int) std::max<int64_t>(1, std::min<int64_t>(all / kSumCtas, p.c.n_max) / kSumKeys) * kSumKeys;
    const int     key_chunks = (p.c.n_max + keys - 1) / keys;
    cfg.gridDim          = dim3((unsigned) (n_out + (p.weight ? p.c.B * p.c.Hkv * key_chunks : 0)));
    cfg.blockDim         = dim3(kSumThreads);
    cfg.dynamicSmemBytes = sizeof(int) * (2 * (size_t) p.c.B + 1);
    return cudaLaunchKernelEx(&cfg, kv8_attn_sum_kernel<HD>, p, 8 * NT, n_out, key_chunks, keys);
}

}  // namespace

// A cluster per unit (in one wave) or runs of tiles over the whole device and
// a second launch?  A CTA's tiles either way, and the second launch with its
// way through HBM as kSecond tiles (0.7 us each; it measured ~3 us).
int kv8_attn_cluster(const Kv8AttnParams &p, int64_t units, int sm_count) {
    constexpr int64_t kSecond = 4;
    const int64_t     nt = (p.c.n_max + kKv8Block - 1) / kKv8Block;
    const int64_t     c  = std::min<int64_t>({8, nt, (int64_t) kCtasPerSm * sm_count / units});
    if (c < 1 || (p.weight && p.n_rb > 1)) {
        return 0;
    }
    const int64_t split = (units * (nt + kUnitCost) + p.n_cta - 1) / p.n_cta;
    return (nt + c - 1) / c <= split + kSecond ? (int) c : 0;
}

int kv8_attn_ctas_per_sm() { return kCtasPerSm; }

int launch_kv8_attn(const Kv8AttnParams &p, cudaStream_t s) {
    CUtensorMap km, vm;
    if (!encode_side(&km, p.c, p.c.k, 64, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        !encode_side(&vm, p.c, p.c.v, p.c.D, p.c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B)) {
        return ACEFA_ERR_LAYOUT;
    }
    const bool one  = p.q.type != ACEFA_TYPE_F32 && p.dst.type != ACEFA_TYPE_F32;
    auto       pick = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (kv8_unit_rows(p.rows, p.q.type) == 16) {
            return one ? launch<HD, 2, kOne>(p, km, vm, s) : launch<HD, 2, kSplit>(p, km, vm, s);
        }
        return one ? launch<HD, 1, kOne>(p, km, vm, s)
                   : (p.rows <= 4 ? launch<HD, 1, kPacked>(p, km, vm, s) : launch<HD, 1, kSplit>(p, km, vm, s));
    };
    const cudaError_t e = p.c.D == 128 ? pick(std::integral_constant<int, 128>{}) : pick(std::integral_constant<int, 64>{});
    return e == cudaSuccess ? ACEFA_OK : ACEFA_ERR_CUDA;
}

}  // namespace acefa
