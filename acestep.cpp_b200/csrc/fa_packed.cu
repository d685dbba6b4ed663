// fa_packed.cu -- attention of whole sequences packed behind one another
// (acefa_flash_attn_packed) on the tensor cores: a persistent tcgen05 / TMEM / TMA
// kernel, described here, and one on mma.sync for few rows further down.
//
// Mathematics: the online softmax in log2 units, S = Q K^T and O += P V on
// 128-row x 128-key tiles with F32 accumulators in tensor memory; P is rounded to
// the operands' type (F16 or BF16), its row sum is not.  A row's maximum only
// moves when it grows by more than 2^8, and O is rescaled only then.  What is
// subtracted lies kLift below that maximum: F16's steps end at 2^-24, and with P from
// 2^15 down only weights below 2^-32 of the row's largest are lost in them (BF16
// has F32's exponents).
//
// Work.  An item is a 128-token tile of one query head; the items of a
// (sequence, KV head), tokens slowest, go two by two to one CTA, which streams
// their keys once for both (with an even number of heads per KV head the two
// are heads of the same tokens, so short sequences waste no second tile).  The
// CTAs are persistent: pairs are numbered from the longest (the last tokens of
// a causal sequence see the most keys) and dealt out back and forth, and the
// warps' pipelines run on across pairs -- the next pair's Q, K and V arrive and
// its first S is computed while this pair's output is still being written.
//   warp 0      TMA: Q (2 x 32 KB) and the key tiles (2 x 32 KB of K and of V).  Tile
//               x's V and tile x + 1's K are awaited and given back together: they
//               serve the same step of the tensor core, and a barrier less per
//               step is time in which it does not run dry.
//   warp 1      MMA issue (one thread); owns TMEM: O0 | O1 | S0 | S1
//   warp 3      finds the CTA's units and hands them to the others through a ring
//   warp 2      where a sequence ends inside a V tile, zeroes its rows behind the
//               end: they belong to other sequences or to nobody, and 0 * NaN is NaN
//   warps 4-7 / 8-11  softmax, rescaling and output of tile 0 / 1, a row per thread
// The rows of Q behind a sequence's end are computed on whatever they hold and
// dropped.  Every wait is bounded (error word and drain on expiry).
//
// Measured (B200): 4096 + 2751 + 1201 causal rows, 16 / 8 heads, D = 128, BF16:
// 119-121 us, 870-890 TFLOP/s of visible pairs, tensor pipe 53 % -- bound by the
// chain S -> softmax -> P -> O of each tile and the issuing thread's waits
// (shared memory feeds the S products at its full 128 B per clock); 16 prompts of
// 64 .. 1024 rows, 32 / 8 heads: 88 us, a third of it the units' beginnings and ends.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "fa_internal.h"
#include "kv8_internal.h"  // find_item, launch_pdl
#include "ptx.cuh"

namespace acefa {
namespace {

struct PackedParams {
    char          *dst;
    int64_t        d_nb1, d_nb2;  // head, row
    const int32_t *cu_q, *cu_k;
    int            n_seq, rows_q, rows_kv, Hkv, G;  // G query heads per KV head
    uint32_t       inv_hkv, inv_g;  // floor(2^32 / d) (d = 1: 2^32 - 1), for divide()
    int            mask, window;
    int            dst_type;
    int            vec;  // output rows are 16-B aligned
    float          scale_log2;
    int           *dev_err;
    uint64_t       wait_limit_ns;
};

constexpr int      kBM = 128, kBN = 128;
constexpr int      kThreads   = 384;
constexpr int      kRing      = 4;
constexpr int      kTileBytes = 128 * 128 * 2;  // 128 rows x 128 dims
constexpr int      kOffRing   = 2 * kTileBytes;  // Q tiles first
constexpr int      kOffBars   = kOffRing + kRing * kTileBytes;
constexpr int      kUnitRing  = 4;                       // units known ahead
constexpr int      kUnitReaders = 11;                    // warps that read them: all but the one that finds them
constexpr int      kNumBars   = 2 * 2 + 2 * 4 + 5 + 2 * kUnitRing;
constexpr int      kOffMisc   = kOffBars + kNumBars * 8;
constexpr int      kOffUnits  = (kOffMisc + 16 + 15) / 16 * 16;
constexpr int      kOffOut    = kOffUnits + kUnitRing * 64;  // where each softmax warp's rows go
constexpr int      kOffStage  = (kOffOut + 8 * 16 + 127) / 128 * 128;  // output rows, 4 KB per softmax warp
constexpr int      kSmemBytes = kOffStage + 8 * 4096 + 1024;  // + alignment of the dynamic base
static_assert(kSmemBytes <= 232448, "more than the 227 KB of a CTA");
constexpr uint32_t kTmemCols  = 512;
constexpr float    kSlack     = 8.0f;
template <bool BF16>
constexpr float kLift = BF16 ? 0.0f : 7.0f;  // with kSlack: P is 2^15 at most, F16 holds 2^16
// Register split (setmaxnreg): the sum must stay within what the block was
// launched with, 384 x 168 = 64512, or setmaxnreg.inc would wait forever.
constexpr uint32_t kRegsControl = 112;
constexpr uint32_t kRegsSoftmax = 192;
static_assert(128 * kRegsControl + 256 * kRegsSoftmax <= 384 * 168, "register split exceeds the launch pool");

// The rows of sequence s; empty and bad for offsets that are none.  Where the
// offsets of Q fall, the sequences behind could meet the rows of those before:
// they end there.
struct Seq {
    int  q0, n_q, k0, n_k;
    bool bad, end;
};
__device__ __forceinline__ Seq seq_of(const PackedParams &P, int s) {
    const int a = P.cu_q[s], b = P.cu_q[s + 1], c = P.cu_k[s], d = P.cu_k[s + 1];
    Seq       r = {a, b - a, c, d - c, false, false};
    if (a < 0 || b < a || b > P.rows_q || c < 0 || d < c || d > P.rows_kv) {
        r = {0, 0, 0, 0, true, b < a};
    }
    return r;
}

// Keys [lo, hi) that query i of the sequence sees; neither end falls as i grows.
__device__ __forceinline__ void visible(const PackedParams &P, const Seq &s, int i, int &lo, int &hi) {
    lo = 0, hi = s.n_k;
    if (P.mask == ACEFA_MASK_CAUSAL) {
        hi = min(max(i + s.n_k - s.n_q + 1, 0), s.n_k);
    } else if (P.mask == ACEFA_MASK_WINDOW) {
        lo = min(max(i - P.window, 0), s.n_k);
        hi = (int) min((int64_t) i + P.window + 1, (int64_t) s.n_k);
    }
}

__device__ __forceinline__ int n_pairs(const PackedParams &P, int n_q) {
    return ((n_q + kBM - 1) / kBM * P.G + 1) >> 1;
}

// n / d with inv = floor(2^32 / d): the product's high word is at most one short.
__device__ __forceinline__ int divide(int n, int d, uint32_t inv) {
    const int q = (int) __umulhi((uint32_t) n, inv);
    return q + (n - q * d >= d);
}

// One CTA's piece of work: up to two items that share a KV head's keys.
struct alignas(16) Unit {
    int q0, n_q, k0, n_k;   // rows of the sequence
    int hk, more;           // KV head; 0: behind the last unit
    int ja, jb;             // key tiles [ja, jb) that some row sees: the tiles' ranges together (they meet)
    int row0[2], head[2];   // first token of a tile in its sequence, its query head
    int a[2], b[2];         // key tiles [a, b) of a tile; row0 >= n_q: no such tile
};
static_assert(sizeof(Unit) == 64, "a slot of the ring");

// The u-th unit (t.more = 0 behind the last); the whole warp gets the same answer.
// Up to 32 sequences (`mine`: lane s holds sequence s) are numbered by length:
// level L holds the pair L of every sequence that has one, the highest first.
// More are numbered one after another, each from its last pair; the search goes
// on from the sequence `from`, before which `before` pairs lie (0, 0 at first:
// a CTA asks for ever higher units, so it passes over the sequences once).
__device__ __forceinline__ void find_unit(const PackedParams &P, int u, const Seq &mine, int &from, int &before, Unit &t) {
    const int x = divide(u, P.Hkv, P.inv_hkv);
    int       pair;
    Seq       q;
    t.hk   = u - x * P.Hkv;
    t.more = 0;
    if (P.n_seq <= 32) {
        const int np = n_pairs(P, mine.n_q);
        if (x >= (int) __reduce_add_sync(0xffffffffu, np)) {
            return;
        }
        // items at level L or above: falls with L; the unit's level is the last with more than x
        int lo = 0, hi = (int) __reduce_max_sync(0xffffffffu, np);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (x < (int) __reduce_add_sync(0xffffffffu, max(np - mid, 0))) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        pair         = lo;
        const int  k = x - (int) __reduce_add_sync(0xffffffffu, max(np - lo - 1, 0));
        // the k-th sequence (from 0) that reaches the level
        const unsigned m    = __ballot_sync(0xffffffffu, np > lo);
        const int      lane = threadIdx.x & 31;
        const int      src  = __ffs(__ballot_sync(0xffffffffu, np > lo && __popc(m & ((1u << lane) - 1u)) == k)) - 1;
        q.q0  = __shfl_sync(0xffffffffu, mine.q0, src);
        q.n_q = __shfl_sync(0xffffffffu, mine.n_q, src);
        q.k0  = __shfl_sync(0xffffffffu, mine.k0, src);
        q.n_k = __shfl_sync(0xffffffffu, mine.n_k, src);
    } else {
        const int lane = threadIdx.x & 31;
        int       np, incl;
        unsigned  hit;
        for (;; from += 32) {
            if (from >= P.n_seq) {
                return;
            }
            const Seq      s   = from + lane < P.n_seq ? seq_of(P, from + lane) : Seq{};
            const unsigned end = __ballot_sync(0xffffffffu, s.end);
            np   = end && lane >= __ffs(end) - 1 ? 0 : n_pairs(P, s.n_q);
            incl = np;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, off);
                incl += lane >= off ? v : 0;
            }
            hit = __ballot_sync(0xffffffffu, x < before + incl);
            if (hit) {
                break;
            }
            if (end) {
                return;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        const int l = __ffs(hit) - 1;
        q    = seq_of(P, from + l);
        pair = __shfl_sync(0xffffffffu, before + incl, l) - 1 - x;
    }
    t.more = 1;
    t.q0 = q.q0, t.n_q = q.n_q, t.k0 = q.k0, t.n_k = q.n_k;
    t.ja = 1 << 30, t.jb = 0;
    const int tt = divide(2 * pair, P.G, P.inv_g), g = 2 * pair - tt * P.G;  // of the first item
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool wrap = i && g + 1 == P.G;
        t.row0[i]       = (tt + (wrap ? 1 : 0)) * kBM;
        t.head[i]       = t.hk * P.G + (wrap ? 0 : g + i);
        t.a[i] = t.b[i] = 0;
        if (t.row0[i] < q.n_q) {
            int lo, hi, unused;
            visible(P, q, t.row0[i], lo, unused);
            visible(P, q, min(t.row0[i] + kBM, q.n_q) - 1, unused, hi);
            if (lo < hi) {
                t.a[i] = lo / kBN, t.b[i] = (hi + kBN - 1) / kBN;
                t.ja = min(t.ja, t.a[i]), t.jb = max(t.jb, t.b[i]);
            }
        }
    }
    t.ja = min(t.ja, t.jb);
}

// Unit number k of this CTA: rounds of gridDim.x units, dealt out back and forth.
__device__ __forceinline__ int deal(int k) {
    return k * (int) gridDim.x + ((k & 1) ? (int) (gridDim.x - 1 - blockIdx.x) : (int) blockIdx.x);
}

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

// Bits [a, b) of a 32-bit word (a, b clipped to 0..32).
__device__ __forceinline__ uint32_t bit_range(int a, int b) {
    a = max(a, 0);
    b = min(b, 32);
    if (a >= b) {
        return 0u;
    }
    return (b >= 32 ? ~0u : ((1u << b) - 1u)) & ~((1u << a) - 1u);
}

__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// The largest of a row's 32 scores and mx; with VIS, keys whose bit of v is 0 become -inf.
template <bool VIS>
__device__ __forceinline__ float max_chunk(uint32_t (&x)[32], uint32_t v, float mx) {
    float m2[2] = {mx, -INFINITY};
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
        if constexpr (VIS) {
            x[e]     = (v >> e) & 1u ? x[e] : 0xFF800000u;
            x[e + 1] = (v >> (e + 1)) & 1u ? x[e + 1] : 0xFF800000u;
        }
        m2[(e >> 1) & 1] = fmax3(m2[(e >> 1) & 1], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
    }
    return fmaxf(m2[0], m2[1]);
}

// P = exp2(x * c - m) of 32 scores, packed two by two over TMEM columns tP .. + 15; sums into ls.
template <bool BF16>
__device__ __forceinline__ void exp_chunk(const uint32_t (&x)[32], uint32_t tP, float c, float m, uint64_t (&ls)[2]) {
    const uint64_t c2 = f32x2(c, c), m2 = f32x2(-m, -m);
    uint32_t       pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float a0, a1;
        f32x2_split(ffma2(f32x2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), c2, m2), a0, a1);
        const float p0 = fast_exp2(a0), p1 = fast_exp2(a1);
        ls[e & 1]      = fadd2(ls[e & 1], f32x2(p0, p1));
        pk[e]          = pack2<BF16>(p0, p1);
    }
    tmem_st16(tP, pk);
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    fa_packed_kernel(const __grid_constant__ PackedParams P, const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t      *smem    = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t     *full    = reinterpret_cast<uint64_t *>(smem + kOffBars);  // [2] V of a tile and K of the next are there
    uint64_t     *empty   = full + 2;
    uint64_t     *s_ready = empty + 2;       // S of tile i is in TMEM
    uint64_t     *p_ready = s_ready + 2;     // P of tile i is in TMEM
    uint64_t     *p_half  = p_ready + 2;     // its first 64 keys are
    uint64_t     *o_done  = p_half + 2;      // O of tile i is complete (once per unit)
    uint64_t     *q_full  = o_done + 2;      // the unit's Q has landed (and the very first K)
    uint64_t     *q_empty = q_full + 1;      // its last S is computed
    uint64_t     *ragged  = q_empty + 1;     // [2] a V tile with rows behind the sequence's end has landed
    uint64_t     *fin     = ragged + 2;
    uint64_t     *u_full  = fin + 1;         // [kUnitRing] a unit is there
    uint64_t     *u_empty = u_full + kUnitRing;
    Unit         *units   = reinterpret_cast<Unit *>(smem + kOffUnits);
    uint32_t     *s_tmem  = reinterpret_cast<uint32_t *>(smem + kOffMisc);
    volatile int *abort_f = reinterpret_cast<volatile int *>(smem + kOffMisc + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 1) {
        tmem_alloc(s_tmem, kTmemCols);
        tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], 2);  // one arrival for V, one for K
            mbar_init(&empty[i], 1);
            mbar_init(&s_ready[i], 1);
            mbar_init(&p_ready[i], 4);  // the tile's warps
            mbar_init(&p_half[i], 4);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(&ragged[0], 1);
        mbar_init(&ragged[1], 1);
        mbar_init(fin, 1);
        for (int i = 0; i < kUnitRing; ++i) {
            mbar_init(&u_full[i], 1);
            mbar_init(&u_empty[i], kUnitReaders);
        }
        *abort_f = 0;
        fence_barrier_init();
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *s_tmem, 0);
    pdl_wait_primary();

    auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
        return mbar_wait_bounded(bar, parity & 1u, abort_f, P.dev_err, code, P.wait_limit_ns);
    };

    // The k-th unit of this CTA, read by a whole warp; false behind the last (or on expiry).
    auto next_unit = [&](int &k, Unit &t) {
        const int  slot = k % kUnitRing;
        const bool ok   = __all_sync(0xffffffffu, wait(&u_full[slot], (uint32_t) (k / kUnitRing), DEVERR_TIMEOUT_FULL));
        t               = units[slot];
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&u_empty[slot]);
        }
        ++k;
        return ok && t.more != 0;
    };

    if (warp < 4) {
        setmaxnreg_dec<kRegsControl>();
        if (warp == 3) {
            // ============================ units ====================================
            Seq mine = {};
            if (P.n_seq <= 32) {
                mine               = lane < P.n_seq ? seq_of(P, lane) : mine;
                const unsigned end = __ballot_sync(0xffffffffu, mine.end);
                mine               = end && lane >= __ffs(end) - 1 ? Seq{} : mine;
            }
            Unit t;
            bool ok   = true;
            int  from = 0, before = 0;
            for (int k = 0; ok; ++k) {
                find_unit(P, deal(k), mine, from, before, t);
                ok = __all_sync(0xffffffffu, wait(&u_empty[k % kUnitRing], (uint32_t) (k / kUnitRing) ^ 1u,
                                                  DEVERR_TIMEOUT_EMPTY));
                if (ok && lane == 0) {
                    units[k % kUnitRing] = t;
                    mbar_arrive(&u_full[k % kUnitRing]);
                }
                ok = ok && t.more != 0;
            }
            for (int s = (int) blockIdx.x * 32 + lane; s < P.n_seq; s += (int) gridDim.x * 32) {
                if (seq_of(P, s).bad) {
                    atomicCAS(P.dev_err, 0, DEVERR_APPEND_POS);
                }
            }
        } else if (warp == 0) {
            // ============================ TMA producer ============================
            // A V tile that ends behind its sequence signals `ragged` of its
            // buffer; warp 2 passes it on to `full` when it is clean.
            int  x = 0, n_unit = 0, n_rag0 = 0, n_rag1 = 0, k = 0;  // x: key tiles so far
            bool ok = true;
            Unit t;
            while (ok && next_unit(k, t)) {
                if (t.ja == t.jb) {
                    continue;
                }
                if (lane == 0) {
                    const bool     two     = t.row0[1] < t.n_q;  // (the first tile is there in every unit)
                    const uint32_t q_bytes = (uint32_t) (kBM * HD * 2) * (two ? 2u : 1u);
                    auto load_k = [&](int j, uint64_t *bar) {
#pragma unroll
                        for (int e = 0; e < HD / 64; ++e) {
                            tma_load_3d(smem + kOffRing + (x & 1) * 2 * kTileBytes + e * (kBN * 128), &kmap, 64 * e,
                                        t.k0 + j * kBN, t.hk, bar);
                        }
                    };
                    if (x > 0) {  // its place was free when the previous V went out
                        mbar_arrive_expect_tx(&full[(x - 1) & 1], kBN * HD * 2);
                        load_k(t.ja, &full[(x - 1) & 1]);
                    }
                    ok = wait(q_empty, (uint32_t) n_unit ^ 1u, DEVERR_TIMEOUT_EMPTY);
                    if (ok) {
                        mbar_arrive_expect_tx(q_full, q_bytes + (x > 0 ? 0u : (uint32_t) (kBN * HD * 2)));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
#pragma unroll
                            for (int h = 0; h < HD / 64; ++h) {
                                if (i == 0 || two) {
                                    tma_load_3d(smem + i * kTileBytes + h * (kBM * 128), &qmap, 64 * h,
                                                t.q0 + t.row0[i], t.head[i], q_full);
                                }
                            }
                        }
                        if (x == 0) {
                            load_k(t.ja, q_full);
                        }
                    }
                    for (int j = t.ja; j < t.jb && ok; ++j) {
                        const int b = x & 1;
                        // (the very first K counts as a pair of its own before empty[1]'s others)
                        ok = wait(&empty[b], (uint32_t) (x >> 1) ^ (b ? 0u : 1u), DEVERR_TIMEOUT_EMPTY);
                        if (!ok) {
                            break;
                        }
                        const bool rag = t.n_k < (j + 1) * kBN;
                        uint64_t  *bar = rag ? &ragged[b] : &full[b];
                        n_rag0 += rag && b == 0;
                        n_rag1 += rag && b == 1;
                        mbar_arrive_expect_tx(bar, kBN * HD * 2);
#pragma unroll
                        for (int e = 0; e < HD / 64; ++e) {
                            tma_load_3d(smem + kOffRing + (2 * b + 1) * kTileBytes + e * (kBN * 128), &vmap, 64 * e,
                                        t.k0 + j * kBN, t.hk, bar);
                        }
                        ++x;
                        if (j + 1 < t.jb) {
                            mbar_arrive_expect_tx(&full[b], kBN * HD * 2);
                            load_k(j + 1, &full[b]);
                        }
                    }
                }
                ++n_unit;
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if (lane == 0 && x > 0) {
                mbar_arrive(&full[(x - 1) & 1]);  // no K goes with the last V
            }
            if (*abort_f && lane == 0) {
                // Let the copies in flight land before the CTA exits: the last of
                // every barrier that this thread announced (one that waits for
                // warp 2 or for a copy never started may stay open; the wait is bounded).
                const uint64_t ts = globaltimer_ns();
                auto drain = [&](uint64_t *bar, int n) {  // n phases announced
                    while (n > 0 && !mbar_try_wait(bar, (uint32_t) (n - 1) & 1u)) {
                        if (globaltimer_ns() - ts > P.wait_limit_ns) {
                            atomicCAS(P.dev_err, 0, DEVERR_TIMEOUT_DRAIN);
                            break;
                        }
                    }
                };
                drain(q_full, n_unit);
                drain(&ragged[0], n_rag0);
                drain(&ragged[1], n_rag1);
                drain(&full[0], (x + 1) >> 1);
                drain(&full[1], x >> 1);
            }
        } else if (warp == 1) {
            // ============================ MMA issuer ==============================
            constexpr uint32_t idS = umma_idesc_f16(128, 128, false, false, BF16);
            constexpr uint32_t idO = umma_idesc_f16(128, HD, false, true, BF16);
            const uint64_t     qd  = umma_desc_sw128(smem_u32(smem), 16, 1024);
            const uint64_t     kd  = umma_desc_sw128(smem_u32(smem + kOffRing), 16, 1024);
            const uint64_t     vd  = umma_desc_sw128(smem_u32(smem + kOffRing), kBN * 128, 1024);
            auto issue_s = [&](int i, int slot) {
                const uint64_t q1 = qd + (uint64_t) (i * (kTileBytes >> 4)), k1 = kd + (uint64_t) (slot * (kTileBytes >> 4));
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint64_t off = (uint64_t) ((ks >> 2) * (kBM * 128 >> 4) + (ks & 3) * 2);
                    umma_ss(tmem + 256 + 128 * i, q1 + off, k1 + off, idS, ks > 0 ? 1u : 0u);
                }
                tc_commit(&s_ready[i]);
            };
            // keys [64 h, 64 h + 64) of the tile
            auto issue_pv = [&](int i, int h, int slot, bool acc) {
                const uint64_t v1 = vd + (uint64_t) (slot * (kTileBytes >> 4));
#pragma unroll
                for (int ks = 4 * h; ks < 4 * h + 4; ++ks) {
                    umma_ts(tmem + 128 * i, tmem + 256 + 128 * i + ks * 8, v1 + (uint64_t) (ks * (16 * 128 >> 4)), idO,
                            ks > 0 || acc ? 1u : 0u);
                }
            };
            // One thread walks the steps (unit, key tile) alone: this loop's own
            // instructions are time in which the tensor core runs dry.
            if (lane == 0) {
                int  k = 0, n_unit = 0;
                bool ok = true;
                Unit t;
                // the next unit with keys; t.more = 0 behind the last or on expiry
                auto enter_unit = [&]() {
                    do {
                        const int slot = k % kUnitRing;
                        ok             = wait(&u_full[slot], (uint32_t) (k / kUnitRing), DEVERR_TIMEOUT_FULL);
                        t              = units[slot];
                        mbar_arrive(&u_empty[slot]);
                        ++k;
                        t.more = ok ? t.more : 0;
                    } while (t.more && t.ja == t.jb);
                };
                auto wait_q = [&]() {
                    ok = ok && wait(q_full, (uint32_t) n_unit, DEVERR_TIMEOUT_FULL);
                    ++n_unit;
                    tc_fence_after();
                };
                auto do_pv = [&](int i, uint32_t ph, int vslot, bool first, bool last) {
                    ok = ok && wait(&p_half[i], ph, DEVERR_TIMEOUT_MMA);
                    tc_fence_after();
                    if (ok) {
                        issue_pv(i, 0, vslot, !first);
                    }
                    ok = ok && wait(&p_ready[i], ph, DEVERR_TIMEOUT_MMA);
                    tc_fence_after();
                    if (ok) {
                        issue_pv(i, 1, vslot, true);
                        if (last) {
                            tc_commit(&o_done[i]);
                        }
                    }
                };
                uint32_t ph0 = 0u, ph1 = 0u;
                int      x = 0;  // key tiles so far; K of tile x is in ring slot 2 * (x & 1), V behind it
                enter_unit();
                int  j = t.ja;
                bool l0 = false, l1 = false;  // tiles that see this key tile
                if (t.more) {
                    l0 = j >= t.a[0] && j < t.b[0], l1 = j >= t.a[1] && j < t.b[1];
                    wait_q();
                    if (ok && l0) {
                        issue_s(0, 0);
                    }
                    if (ok && l1) {
                        issue_s(1, 0);
                    }
                    tc_commit(&empty[1]);
                    if (j + 1 == t.jb) {
                        tc_commit(q_empty);
                    }
                }
                while (ok && t.more) {
                    const bool f0 = j == t.a[0], f1 = j == t.a[1], e0 = j + 1 == t.b[0], e1 = j + 1 == t.b[1];
                    const int  b = x & 1, vslot = 2 * b + 1, kslot = 2 * (b ^ 1);
                    ++j;
                    const bool new_q = j == t.jb;
                    if (new_q) {
                        enter_unit();
                        j = t.ja;
                    }
                    const bool more = t.more != 0;
                    const bool n0   = more && j >= t.a[0] && j < t.b[0], n1 = more && j >= t.a[1] && j < t.b[1];
                    ok = ok && wait(&full[b], (uint32_t) (x >> 1), DEVERR_TIMEOUT_FULL);
                    tc_fence_after();
                    if (!new_q) {
                        // S of the next step between the tiles' PVs
                        if (l0) {
                            do_pv(0, ph0, vslot, f0, e0);
                            ph0 ^= 1u;
                        }
                        if (ok && n0) {
                            issue_s(0, kslot);
                        }
                        if (l1) {
                            do_pv(1, ph1, vslot, f1, e1);
                            ph1 ^= 1u;
                        }
                        if (ok && n1) {
                            issue_s(1, kslot);
                        }
                    } else {
                        // the end of a unit: the next one's S waits for its Q, so both PVs go first
                        if (l0) {
                            do_pv(0, ph0, vslot, f0, e0);
                            ph0 ^= 1u;
                        }
                        if (l1) {
                            do_pv(1, ph1, vslot, f1, e1);
                            ph1 ^= 1u;
                        }
                        if (more) {
                            wait_q();
                            if (ok && n0) {
                                issue_s(0, kslot);
                            }
                            if (ok && n1) {
                                issue_s(1, kslot);
                            }
                        }
                    }
                    tc_commit(&empty[b]);
                    if (more && j + 1 == t.jb) {
                        tc_commit(q_empty);
                    }
                    l0 = n0, l1 = n1;
                    ++x;
                }
            }
            if (lane == 0) {
                // every MMA issued by this thread completes before TMEM is released
                tc_commit(fin);
                const uint64_t ts = globaltimer_ns();
                while (!mbar_try_wait(fin, 0)) {
                    if (globaltimer_ns() - ts > P.wait_limit_ns) {
                        atomicCAS(P.dev_err, 0, DEVERR_TIMEOUT_MMA);
                        break;
                    }
                }
            }
        } else if (warp == 2) {
            // ==================== V rows behind the sequence's end =================
            int  x = 0, n_rag0 = 0, n_rag1 = 0, k = 0;
            bool ok = true;
            Unit t;
            while (ok && next_unit(k, t)) {
                x += t.jb - t.ja;
                if (t.ja < t.jb && t.n_k < t.jb * kBN) {
                    const int b = (x - 1) & 1;  // the unit's last tile
                    ok = __all_sync(0xffffffffu, wait(&ragged[b], (uint32_t) (b ? n_rag1 : n_rag0), DEVERR_TIMEOUT_FULL));
                    n_rag0 += b == 0;
                    n_rag1 += b == 1;
                    if (ok) {
                        // a row is 128 contiguous bytes of each 64-dim box (the swizzle stays inside them)
                        const int valid = t.n_k - (t.jb - 1) * kBN;
#pragma unroll
                        for (int e = 0; e < HD / 64; ++e) {
                            uint4 *p = reinterpret_cast<uint4 *>(smem + kOffRing + (2 * b + 1) * kTileBytes + e * (kBN * 128));
                            for (int y = valid * 8 + lane; y < kBN * 8; y += 32) {
                                p[y] = make_uint4(0u, 0u, 0u, 0u);
                            }
                        }
                        fence_proxy_async_smem();  // read next by the tensor core
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&full[b]);
                        }
                    }
                }
            }
        }
    } else {
        // ============================ softmax =================================
        setmaxnreg_inc<kRegsSoftmax>();
        const int      i     = (warp - 4) >> 2;  // tile
        const int      r     = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16;
        const uint32_t tS    = tmem + lanes + 256 + 128 * i;
        const uint32_t tO    = tmem + lanes + 128 * i;
        const float    c     = P.scale_log2;
        uint32_t       n_s = 0, n_o = 0;  // S tiles and finished units so far
        bool           ok = true;
        int            k  = 0;
        uint8_t       *stage = smem + kOffStage + (warp - 4) * 4096;
        volatile int  *out_at = reinterpret_cast<volatile int *>(smem + kOffOut) + (warp - 4) * 4;
        Unit           t;
        while (ok && next_unit(k, t)) {
            // (selects, not an index: the unit stays in registers)
            const int row0 = i ? t.row0[1] : t.row0[0], head = i ? t.head[1] : t.head[0];
            const int ja = i ? t.a[1] : t.a[0], jb = i ? t.b[1] : t.b[0];
            if (row0 >= t.n_q) {
                continue;
            }
            const Seq  q        = {t.q0, t.n_q, t.k0, t.n_k, false, false};
            const int  row      = row0 + r;
            const bool mine_row = row < q.n_q;
            int        vlo = 0, vhi = 0;
            if (mine_row) {
                visible(P, q, row, vlo, vhi);
            }
            // keys that every row of the tile sees: such key tiles need no masks
            int all_lo, all_hi, unused;
            visible(P, q, min(row0 + kBM, q.n_q) - 1, all_lo, unused);
            visible(P, q, row0, unused, all_hi);
            // what the output needs waits in shared memory: the loop's registers are full of scores
            if (lane == 0) {
                const int w0 = row0 + (warp & 3) * 32;  // the warp's first row
                out_at[0] = q.q0 + w0, out_at[1] = q.n_q - w0, out_at[2] = head;
            }
            __syncwarp();
            // rows behind the sequence's end: under +inf their weights are 0 and their maximum never moves
            float m_run = mine_row ? -INFINITY : INFINITY, l_run = 0.0f;
            for (int j = ja; j < jb && ok; ++j) {
                const int  j0   = j * kBN;
                const bool open = j0 >= all_lo && j0 + kBN <= all_hi;
                ok = __all_sync(0xffffffffu, wait(&s_ready[i], n_s, DEVERR_TIMEOUT_MMA));
                ++n_s;
                if (!ok) {
                    break;
                }
                tc_fence_after();
                // the row's scores stay in registers between the maximum and the exponentials
                uint32_t x0[32], x1[32], x2[32], x3[32];
                tmem_ld32(tS, x0);
                tmem_ld32(tS + 32, x1);
                tmem_ld32(tS + 64, x2);
                tmem_ld32(tS + 96, x3);
                tmem_ld_wait32(x0);
                tmem_ld_wait32(x1);
                tmem_ld_wait32(x2);
                tmem_ld_wait32(x3);
                float top = -INFINITY;
                if (open) {
                    top = max_chunk<false>(x0, 0u, top);
                    top = max_chunk<false>(x1, 0u, top);
                    top = max_chunk<false>(x2, 0u, top);
                    top = max_chunk<false>(x3, 0u, top);
                } else {
                    top = max_chunk<true>(x0, bit_range(vlo - j0, vhi - j0), top);
                    top = max_chunk<true>(x1, bit_range(vlo - j0 - 32, vhi - j0 - 32), top);
                    top = max_chunk<true>(x2, bit_range(vlo - j0 - 64, vhi - j0 - 64), top);
                    top = max_chunk<true>(x3, bit_range(vlo - j0 - 96, vhi - j0 - 96), top);
                }
                top *= c;
                // the first visible key counts: any number is above -inf
                const bool grew = top > m_run + (kSlack + kLift<BF16>);
                if (__any_sync(0xffffffffu, grew)) {
                    const float mn = top - kLift<BF16>;
                    const float f  = grew ? fast_exp2(m_run - mn) : 1.0f;
                    m_run          = grew ? mn : m_run;
                    l_run *= f;
                    if (j > ja) {
#pragma unroll 1
                        for (int ch = 0; ch < HD / 16; ++ch) {
                            uint32_t x[16];
                            tmem_ld16(tO + 16 * ch, x);
                            tmem_ld_wait16(x);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
                            }
                            tmem_st16(tO + 16 * ch, x);
                        }
                    }
                }
                const float m_use = m_run == -INFINITY ? 0.0f : m_run;
                uint64_t    ls[2] = {0ull, 0ull};
                exp_chunk<BF16>(x0, tS, c, m_use, ls);
                exp_chunk<BF16>(x1, tS + 16, c, m_use, ls);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_half[i]);  // the product with V starts on these 64 keys
                }
                exp_chunk<BF16>(x2, tS + 32, c, m_use, ls);
                exp_chunk<BF16>(x3, tS + 48, c, m_use, ls);
                float l0, l1;
                f32x2_split(fadd2(ls[0], ls[1]), l0, l1);
                l_run += l0 + l1;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_ready[i]);
                }
            }
            // ---- O / l leaves: 128-B pieces of the warp's 32 rows through its
            // staging slab (16-B chunk x of row y at x ^ (y & 7): no bank conflicts
            // either way), so that a store instruction writes whole lines
            // (a tile that saw no key reads what O happens to hold, and writes zeros)
            if (ok && ja < jb) {
                ok = __all_sync(0xffffffffu, wait(&o_done[i], n_o, DEVERR_TIMEOUT_MMA));
                ++n_o;
                tc_fence_after();
            }
            if (!ok) {
                break;
            }
            // (opaque copies: their addresses must not be hoisted into the key loop)
            int      ln   = lane;
            uint32_t slab = smem_u32(stage);
            int64_t  nb2  = P.d_nb2;
            asm volatile("" : "+r"(ln), "+r"(slab), "+l"(nb2));
            const bool  none = l_run == 0.0f;  // the row saw nothing: 0, whatever 0 * V has left in O
            const float inv  = none ? 0.0f : 1.0f / l_run;
            const int   rows = out_at[1];  // of this warp, if below 32
            char *out = P.dst + (int64_t) out_at[2] * P.d_nb1 + (int64_t) out_at[0] * nb2;
            // 32 dims of the row, finished
            auto finished = [&](uint32_t(&x)[32]) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    x[e] = __float_as_uint(__uint_as_float(x[e]) * inv);
                }
                if (__any_sync(0xffffffffu, none)) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        x[e] = none ? 0u : x[e];
                    }
                }
            };
            // the slab's 32 x 128 B to dst, piece n of the rows
            auto write_slab = [&](int n, bool f32) {
                __syncwarp();
                uint4 w[8];
#pragma unroll
                for (int st = 0; st < 8; ++st) {
                    const int rr = 4 * st + (ln >> 3);
                    w[st] = ld_shared_v4(slab + rr * 128 + (((ln & 7) ^ (rr & 7)) << 4));
                }
                char *p = out + 128 * n + 16 * (ln & 7) + (int64_t) (ln >> 3) * nb2;
                if (P.vec) {
#pragma unroll
                    for (int st = 0; st < 8; ++st) {
                        if (4 * st + (ln >> 3) < rows) {
                            *reinterpret_cast<uint4 *>(p + (int64_t) (4 * st) * nb2) = w[st];
                        }
                    }
                } else {
#pragma unroll
                    for (int st = 0; st < 8; ++st) {
                        const uint32_t y[4] = {w[st].x, w[st].y, w[st].z, w[st].w};
                        if (4 * st + (ln >> 3) < rows) {
                            for (int e = 0; e < 4; ++e) {
                                char *pe = p + (int64_t) (4 * st) * nb2 + 4 * e;
                                if (f32) {
                                    *reinterpret_cast<uint32_t *>(pe) = y[e];
                                } else {
                                    reinterpret_cast<uint16_t *>(pe)[0] = (uint16_t) y[e];
                                    reinterpret_cast<uint16_t *>(pe)[1] = (uint16_t) (y[e] >> 16);
                                }
                            }
                        }
                    }
                }
                __syncwarp();  // the slab has been read
            };
            uint32_t x[2][32];
            tmem_ld32(tO, x[0]);
            tmem_ld32(tO + 32, x[1]);
#pragma unroll
            for (int n = 0; n < HD / 64; ++n) {  // 64 dims at a time
                tmem_ld_wait32(x[0]);
                tmem_ld_wait32(x[1]);
                finished(x[0]);
                finished(x[1]);
                if (P.dst_type == ACEFA_TYPE_F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            st_shared_v4(slab + ln * 128 + ((e ^ (ln & 7)) << 4), x[h][4 * e], x[h][4 * e + 1],
                                         x[h][4 * e + 2], x[h][4 * e + 3]);
                        }
                        write_slab(2 * n + h, true);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t y[4];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int d = 8 * (e & 3) + 2 * w;
                            y[w] = pack2<BF16>(__uint_as_float(x[e >> 2][d]), __uint_as_float(x[e >> 2][d + 1]));
                        }
                        st_shared_v4(slab + ln * 128 + ((e ^ (ln & 7)) << 4), y[0], y[1], y[2], y[3]);
                    }
                }
                if (n + 1 < HD / 64) {  // on their way while this piece is written
                    tmem_ld32(tO + 64, x[0]);
                    tmem_ld32(tO + 96, x[1]);
                }
                if (P.dst_type != ACEFA_TYPE_F32) {
                    write_slab(n, false);
                }
            }
            tc_fence_before();  // O has been read before the next unit's P is announced
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------------------
// Few rows: the same attention on mma.sync, 16 tokens of one query head per CTA.
// No tensor memory, no staging and no pipeline to fill: each of the four warps takes
// 16 keys of every 64 and loads exactly its fragments' 16-B pieces of rows to
// registers, products run transposed (S^T = K Q^T, O^T = V^T P^T; P changes layout by
// movmatrix), and the warps' results meet once in shared memory.  Bound by latency:
// 2.7-4.4 us up to 128 rows of 16 heads, where the kernel above takes 7.9.
constexpr int   kSmallRows = 16;
constexpr int   kSmallWarps = 4;
constexpr float kNoMax = -1.7e38f;  // below every score, finite

struct SmallParams {
    PackedParams p;
    const char  *q, *k, *v;
    int64_t      q_nb1, q_nb2, k_nb1, k_nb2, v_nb1, v_nb2;  // row, head
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(32 * kSmallWarps) fa_packed_small(const __grid_constant__ SmallParams S) {
    constexpr int NT = kSmallRows / 8, KS = HD / 16, kOut = HD + 4;
    __shared__ float s_o[kSmallWarps][kSmallRows][kOut];
    __shared__ float s_m[kSmallWarps][kSmallRows], s_l[kSmallWarps][kSmallRows];
    pdl_wait_primary();
    const PackedParams &P = S.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int h = blockIdx.y, hk = divide(h, P.G, P.inv_g);
    if (h == 0 && warp == 0) {
        for (int s = (int) blockIdx.x * 32 + lane; s < P.n_seq; s += (int) gridDim.x * 32) {
            if (seq_of(P, s).bad) {
                atomicCAS(P.dev_err, 0, DEVERR_APPEND_POS);
            }
        }
    }
    int si, item;
    auto tiles = [&](int i) {
        const Seq s = seq_of(P, i);
        return s.end ? -1 : (s.n_q + kSmallRows - 1) / kSmallRows;
    };
    if (!find_item(P.n_seq, blockIdx.x, tiles, si, item)) {
        return;
    }
    const Seq q    = seq_of(P, si);
    const int row0 = item * kSmallRows, n_row = min(kSmallRows, q.n_q - row0);
    // ---- Q^T: row nt * 8 + g; the dims of word pairs as K's pieces have them
    uint32_t qf[NT][KS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int   r = nt * 8 + g;
        const char *p = S.q + (int64_t) (q.q0 + row0 + r) * S.q_nb1 + h * S.q_nb2 + 16 * c;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
            const uint4 w = r < n_row ? *reinterpret_cast<const uint4 *>(p + 64 * e) : make_uint4(0u, 0u, 0u, 0u);
            qf[nt][2 * e][0] = w.x, qf[nt][2 * e][1] = w.y, qf[nt][2 * e + 1][0] = w.z, qf[nt][2 * e + 1][1] = w.w;
        }
    }
    int   lo[NT][2], hi[NT][2];  // what rows nt * 8 + 2c, + 1 see
    float m[NT][2], l[NT][2], acc[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * c + e;
            lo[nt][e] = hi[nt][e] = 0;
            if (r < n_row) {
                visible(P, q, row0 + r, lo[nt][e], hi[nt][e]);
            }
            m[nt][e] = kNoMax;
            l[nt][e] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            acc[nt][t][0] = acc[nt][t][1] = acc[nt][t][2] = acc[nt][t][3] = 0.0f;
        }
    }
    int j_lo, j_hi, unused;
    visible(P, q, row0, j_lo, unused);
    visible(P, q, row0 + n_row - 1, unused, j_hi);
    const char *kb = S.k + (int64_t) q.k0 * S.k_nb1 + hk * S.k_nb2 + 16 * c;
    const char *vb = S.v + (int64_t) q.k0 * S.v_nb1 + hk * S.v_nb2 + (HD / 4) * g;
#pragma unroll 1
    for (int j0 = (j_lo & ~15) + 16 * warp; j0 < j_hi; j0 += 16 * kSmallWarps) {
        // K rows g and g + 8, pieces c; V rows 2c, 2c + 1, 2c + 8, 2c + 9, HD / 8 dims
        // of g.  Rows behind the sequence's end are zeros.
        uint4 kw[2][HD / 32], vw[4][HD / 64];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int j = j0 + g + 8 * r;
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) {
                kw[r][e] = j < q.n_k ? *reinterpret_cast<const uint4 *>(kb + j * S.k_nb1 + 64 * e)
                                     : make_uint4(0u, 0u, 0u, 0u);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int j = j0 + 2 * c + (r & 1) + 8 * (r >> 1);
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
                vw[r][e] = j < q.n_k ? *reinterpret_cast<const uint4 *>(vb + j * S.v_nb1 + 16 * e)
                                     : make_uint4(0u, 0u, 0u, 0u);
            }
        }
        // ---- S^T: (key g, rows 2c 2c+1), (key g + 8, the same rows); even and odd k-steps apart
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[nt][e] = s2[nt][e] = 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
            const uint32_t a[4] = {kw[0][e].x, kw[1][e].x, kw[0][e].y, kw[1][e].y};
            const uint32_t b[4] = {kw[0][e].z, kw[1][e].z, kw[0][e].w, kw[1][e].w};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma_16816<BF16>(s[nt], a, qf[nt][2 * e][0], qf[nt][2 * e][1]);
                mma_16816<BF16>(s2[nt], b, qf[nt][2 * e + 1][0], qf[nt][2 * e + 1][1]);
            }
        }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int   j = j0 + g + 8 * (e >> 1);
                const float v = (s[nt][e] + s2[nt][e]) * P.scale_log2;
                s[nt][e]      = j >= lo[nt][e & 1] && j < hi[nt][e & 1] ? v : -INFINITY;
                grow |= s[nt][e] > m[nt][e & 1] + (kSlack + kLift<BF16>);
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
                    const float mn = fmaxf(m[nt][e], top - kLift<BF16>), f = fast_exp2(m[nt][e] - mn);
                    m[nt][e] = mn;
                    l[nt][e] *= f;
#pragma unroll
                    for (int t = 0; t < KS; ++t) {
                        acc[nt][t][e] *= f;
                        acc[nt][t][2 + e] *= f;
                    }
                }
            }
        }
        uint32_t ph[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = fast_exp2(s[nt][e] - m[nt][e & 1]);
                l[nt][e & 1] += p[e];
            }
            ph[nt][0] = movmatrix_trans(pack2<BF16>(p[0], p[1]));
            ph[nt][1] = movmatrix_trans(pack2<BF16>(p[2], p[3]));
        }
        // ---- O^T: m-tile t is dims g * HD / 8 + 2t (row g) and + 2t + 1 (row g + 8)
        uint32_t vr[4][HD / 16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
                vr[r][4 * e] = vw[r][e].x, vr[r][4 * e + 1] = vw[r][e].y;
                vr[r][4 * e + 2] = vw[r][e].z, vr[r][4 * e + 3] = vw[r][e].w;
            }
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            const uint32_t a[4] = {__byte_perm(vr[0][t], vr[1][t], 0x5410u), __byte_perm(vr[0][t], vr[1][t], 0x7632u),
                                   __byte_perm(vr[2][t], vr[3][t], 0x5410u), __byte_perm(vr[2][t], vr[3][t], 0x7632u)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma_16816<BF16>(acc[nt][t], a, ph[nt][0], ph[nt][1]);
            }
        }
    }
    // ---- the warps' results together
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
                s_m[warp][row] = m[nt][e];
                s_l[warp][row] = sum;
            }
#pragma unroll
            for (int t = 0; t < KS; t += 2) {
                *reinterpret_cast<float4 *>(&s_o[warp][row][g * (HD / 8) + 2 * t]) =
                    make_float4(acc[nt][t][e], acc[nt][t][2 + e], acc[nt][t + 1][e], acc[nt][t + 1][2 + e]);
            }
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < n_row * (HD / 4); x += 32 * kSmallWarps) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float     M = kNoMax, L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kSmallWarps; ++w) {
            M = fmaxf(M, s_m[w][r]);
        }
#pragma unroll
        for (int w = 0; w < kSmallWarps; ++w) {
            const float  f = exp2f(s_m[w][r] - M);
            const float4 v = *reinterpret_cast<const float4 *>(&s_o[w][r][d]);
            L = fmaf(s_l[w][r], f, L);
            o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]), o[2] = fmaf(v.z, f, o[2]), o[3] = fmaf(v.w, f, o[3]);
        }
        const float inv = 1.0f / L;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] = L == 0.0f ? 0.0f : o[e] * inv;  // a row that saw nothing is 0
        }
        char *p = P.dst + h * P.d_nb1 + (int64_t) (q.q0 + row0 + r) * P.d_nb2;
        if (P.dst_type == ACEFA_TYPE_F32) {
            float *f = reinterpret_cast<float *>(p) + d;
            if (P.vec) {
                *reinterpret_cast<float4 *>(f) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                f[0] = o[0], f[1] = o[1], f[2] = o[2], f[3] = o[3];
            }
        } else {
            const uint32_t w[2] = {pack2<BF16>(o[0], o[1]), pack2<BF16>(o[2], o[3])};
            uint16_t      *f    = reinterpret_cast<uint16_t *>(p) + d;
            if (P.vec) {
                *reinterpret_cast<uint2 *>(f) = make_uint2(w[0], w[1]);
            } else {
                f[0] = (uint16_t) w[0], f[1] = (uint16_t) (w[0] >> 16);
                f[2] = (uint16_t) w[1], f[3] = (uint16_t) (w[1] >> 16);
            }
        }
    }
}

template <int HD, bool BF16>
cudaError_t launch(const PackedParams &p, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, int n_cta,
                   cudaStream_t s) {
    static thread_local int configured = -1;
    int                     dev        = 0;
    cudaGetDevice(&dev);
    if (configured != dev) {
        cudaError_t e =
            cudaFuncSetAttribute(fa_packed_kernel<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) {
            return e;
        }
        configured = dev;
    }
    return launch_pdl(fa_packed_kernel<HD, BF16>, dim3((unsigned) n_cta), kThreads, kSmemBytes, s, p, q, k, v);
}

// [D, rows, heads] of 16-bit elements, tiles of 64 dims x 128 rows, 128-B swizzle.
int encode_rows(CUtensorMap *map, const acefa_tensor *t) {
    EncodeTiledFn enc = tensor_map_encoder();
    if (!enc) {
        return ACEFA_ERR_CUDA;
    }
    // strides of extent-1 dims do not matter; keep them 16-B multiples
    const cuuint64_t rows = (cuuint64_t) t->ne[1], heads = (cuuint64_t) t->ne[2];
    const cuuint64_t s1   = rows > 1 ? (cuuint64_t) t->nb[1] : 2u * (cuuint64_t) t->ne[0];
    const cuuint64_t s2   = heads > 1 ? (cuuint64_t) t->nb[2] : s1 * rows;
    cuuint64_t       dims[3] = {(cuuint64_t) t->ne[0], rows, heads}, strides[2] = {s1, s2};
    cuuint32_t       box[3] = {64, 128, 1}, estr[3] = {1, 1, 1};
    CUresult rc = enc(map, t->type == ACEFA_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                      3, t->data, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? ACEFA_OK : ACEFA_ERR_LAYOUT;
}

// The few-rows kernel?  It reads the keys again for every 16 rows of a head, so
// its time grows with rows x heads x D; the tensor-memory kernel starts slowly.
// Measured, few-rows against the other (us, causal, BF16, 100 calls in a graph): one
// sequence of 1 / 16 / 128 / 256 rows, 16 heads, D = 128: 2.7 : 7.9, 3.3 : 7.8, 4.4 : 7.9, 7.4 : 9.9;
// 512 rows, 8 / 16 heads: 10.9 : 13.4, 18.0 : 13.4; 256 rows, 32 heads: 12.5 : 10.1; 8 sequences of 578
// rows in all, 8 / 16 heads: 7.7 : 9.7, 11.3 : 10.4; 512 rows, 16 heads, D = 64: 10.4 : 12.0; at the
// rule's edge, 375 rows of 16 heads: 12.6 : 11.8.
bool use_small(int64_t rows_q, int64_t rows_kv, int64_t Hq, int64_t D, int n_seq) {
    return rows_q * Hq * D <= 6000 * 128 && rows_kv <= 1024 && n_seq <= 1024;
}

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// The rows of a tensor on the host: `rows` x `heads` pieces of `bytes`.
struct Pieces {
    int64_t at, bytes, rows, row_nb, heads, head_nb;

    int64_t end() const { return at + (rows - 1) * row_nb + (heads - 1) * head_nb + bytes; }
};

// Whether a and b share an address.  Tensors whose rows are the same distance
// apart may lie in one buffer (the projections of a row and its output behind one
// another); with other distances their extents have to be apart.
bool meet(Pieces a, Pieces b) {
    if (!a.rows || !b.rows || a.at >= b.end() || b.at >= a.end()) {
        return false;
    }
    a.row_nb = a.rows > 1 ? a.row_nb : b.row_nb;
    b.row_nb = b.rows > 1 ? b.row_nb : a.row_nb;
    if (a.row_nb != b.row_nb) {
        return true;
    }
    const int64_t step = a.rows > 1 || b.rows > 1 ? a.row_nb : 1ll << 62;
    auto          floor_div = [](int64_t n, int64_t d) { return n / d - (n % d < 0); };
    for (int64_t i = 0; i < a.heads; ++i) {
        for (int64_t j = 0; j < b.heads; ++j) {
            // row r of a meets row r + d of b where d * step lies in (gap - b.bytes, gap + a.bytes)
            const int64_t gap = a.at + i * a.head_nb - b.at - j * b.head_nb;
            const int64_t lo  = std::max(floor_div(gap - b.bytes, step) + 1, 1 - a.rows);
            const int64_t hi  = std::min(-floor_div(-(gap + a.bytes), step) - 1, b.rows - 1);
            if (lo <= hi) {
                return true;
            }
        }
    }
    return false;
}

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
        if (t->nb[0] != 2 || !aligned(t->data, 16)) {
            return ACEFA_ERR_LAYOUT;
        }
        for (int i = 1; i < 3; ++i) {  // (no tensor map has a stride of 0)
            if (t->ne[i] > 1 && (t->nb[i] % 16 || t->nb[i] == 0)) {
                return ACEFA_ERR_LAYOUT;
            }
        }
    }
    const size_t es = dst->type == ACEFA_TYPE_F32 ? 4 : 2;
    if ((rows_q && (dst->nb[0] != es || !aligned(dst->data, es))) || (Hq > 1 && dst->nb[1] % es) ||
        (rows_q > 1 && dst->nb[2] % es) || !aligned(cu_q, 4) || !aligned(cu_k, 4)) {
        return ACEFA_ERR_LAYOUT;
    }
    // no two rows of dst on one another (its heads and rows in either order)
    const size_t row = (size_t) D * es, heads = dst->nb[1], rows = dst->nb[2];
    if ((Hq > 1 && heads < row) || (rows_q > 1 && rows < row) ||
        (Hq > 1 && rows_q > 1 && rows < heads * (size_t) Hq && heads < rows * (size_t) rows_q)) {
        return ACEFA_ERR_LAYOUT;
    }
    // nor on the rows of q, k and v
    const Pieces out = {(int64_t) (uintptr_t) dst->data, (int64_t) row, rows_q, (int64_t) rows, Hq, (int64_t) heads};
    for (const acefa_tensor *t : {q, k, v}) {
        if (meet(out, {(int64_t) (uintptr_t) t->data, 2 * D, t->ne[1], (int64_t) t->nb[1], t->ne[2], (int64_t) t->nb[2]})) {
            return ACEFA_ERR_LAYOUT;
        }
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
    p.dst   = static_cast<char *>(dst->data);
    p.d_nb1 = (int64_t) dst->nb[1], p.d_nb2 = (int64_t) dst->nb[2];
    p.cu_q = cu_q, p.cu_k = cu_k ? cu_k : cu_q;
    p.n_seq = n_seq, p.rows_q = (int) rows_q, p.rows_kv = (int) rows_kv;
    p.Hkv = (int) Hkv, p.G = (int) (Hq / Hkv);
    auto inverse = [](int d) { return d == 1 ? 0xFFFFFFFFu : (uint32_t) ((1ull << 32) / (uint64_t) d); };
    p.inv_hkv = inverse(p.Hkv), p.inv_g = inverse(p.G);
    p.mask = mask, p.window = window;
    p.dst_type      = dst->type;
    p.vec           = ((reinterpret_cast<uintptr_t>(dst->data) | dst->nb[1] | dst->nb[2]) & 15u) == 0;
    p.scale_log2    = scale * kLog2e;
    p.dev_err       = ctx.dev_err;
    p.wait_limit_ns = ctx.wait_limit_ns;
    const bool bf     = q->type == ACEFA_TYPE_BF16;
    auto       cs = static_cast<cudaStream_t>(stream);
    if (use_small(rows_q, rows_kv, Hq, D, n_seq)) {
        SmallParams sp;
        sp.p = p;
        sp.q = static_cast<const char *>(q->data), sp.k = static_cast<const char *>(k->data);
        sp.v = static_cast<const char *>(v->data);
        sp.q_nb1 = (int64_t) q->nb[1], sp.q_nb2 = (int64_t) q->nb[2];
        sp.k_nb1 = (int64_t) k->nb[1], sp.k_nb2 = (int64_t) k->nb[2];
        sp.v_nb1 = (int64_t) v->nb[1], sp.v_nb2 = (int64_t) v->nb[2];
        const dim3 grid((unsigned) (rows_q / kSmallRows + n_seq), (unsigned) Hq);
        auto       kern = D == 128 ? (bf ? fa_packed_small<128, true> : fa_packed_small<128, false>)
                                   : (bf ? fa_packed_small<64, true> : fa_packed_small<64, false>);
        if (launch_pdl(kern, grid, 32 * kSmallWarps, 0, cs, sp) != cudaSuccess) {
            return ACEFA_ERR_CUDA;
        }
        note_launches(1, 3);
        return ACEFA_OK;
    }
    // no keys at all: nothing is loaded, but the kernel's parameters still want a map
    CUtensorMap qm, km, vm;
    int         mrc = encode_rows(&qm, q);
    if (mrc == ACEFA_OK) {
        mrc = encode_rows(&km, rows_kv ? k : q);
    }
    if (mrc == ACEFA_OK) {
        mrc = encode_rows(&vm, rows_kv ? v : q);
    }
    if (mrc != ACEFA_OK) {
        return mrc;
    }
    // units: at most (tiles of all sequences * G + 1 per sequence) / 2 per KV head
    const int64_t tiles = rows_q / kBM + n_seq;
    const int64_t units = (tiles * (Hq / Hkv) + n_seq) / 2 * Hkv;
    const int     n_cta = (int) std::min<int64_t>(std::max<int64_t>(units, 1), ctx.sm_count);
    cudaError_t   e     = D == 128 ? (bf ? launch<128, true>(p, qm, km, vm, n_cta, cs) : launch<128, false>(p, qm, km, vm, n_cta, cs))
                                   : (bf ? launch<64, true>(p, qm, km, vm, n_cta, cs) : launch<64, false>(p, qm, km, vm, n_cta, cs));
    if (e != cudaSuccess) {
        return ACEFA_ERR_CUDA;
    }
    note_launches(1, 3);
    return ACEFA_OK;
}
