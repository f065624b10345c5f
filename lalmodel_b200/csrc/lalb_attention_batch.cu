// lalb_attention_batch.cu -- one decode step of attention for a batch of
// sequences that share a prefix (lalb_attention_batch), attention_forward
// (runtime/lal_runtime.c:833-882) for many sequences at once.
//
//   out = sum_j 2^(x_j - M) v_j / sum_j 2^(x_j - M),  x_j = (scale log2 e) q . k_j
//
// over the prefix rows and the sequence's own.  Any set of rows j gives a
// partial (m, l, O): a reference exponent m, l = sum_j 2^(x_j - m) and
// O = sum_j 2^(x_j - m) v_j; partials over disjoint sets combine exactly.
//
// Units.  A prefix unit is a KV head and up to 128 query rows of ALL sequences
// (row = sequence * group + head of the group) over the prefix, so its K and V
// are read once for 128 rows instead of once per sequence.  An own unit is one
// sequence's group of heads over its own rows.  Both are the same work: S =
// Q K^T and O += P V with M = 128 rows on tcgen05, 64 cache rows (a tile) at a
// time; an own unit fills only its group's lanes of the M = 128 instructions,
// which costs tensor time that a memory-bound unit has to spare.
//
// Units of at most 16 rows (few sequences, and the own units of all common head
// layouts) leave three of four softmax warps without a row.  Where the softmax
// is what such a unit waits for (Cfg::kFewOk), its Q is written four times, once
// to each warp's 32 lanes, and warp w takes only scores 16 w .. 16 w + 15 of a
// tile, with zeros as the weights of the rest; the four warps' sums are added
// at the segment's end.
//
// Split.  All tiles of all units form one list (List), and every CTA, one per
// SM, takes an equal run of it: equal shares whatever the lengths, without the
// host knowing them.  A run of tiles of one unit in one CTA (a segment) ends in
// one partial; attention_combine_kernel adds a row's partials in list order, so
// results do not depend on scheduling.
//
// One CTA, warp-specialised (kSoftWarps softmax, 1 MMA, the loaders):
//   loaders  K and V tiles into a ring, in the order K0 V0 K1 V1 ..; 16-bit
//            caches by tiled TMA straight into the swizzled operand layout;
//            F32 rows by TMA to the seven loader warps, which split each value
//            into two fp16 parts;
//   MMA      S runs kAhead tiles ahead of PV, so that the tensor cores work on
//            the next scores while the softmax of this tile runs; Q is the A
//            operand from TMEM, P overwrites its S in TMEM as the next A;
//   softmax  two warpgroups on alternate tiles, each with its own O (128 rows
//            = TMEM lanes = threads, so rows need no shuffles); O is rescaled
//            only when a row's maximum has grown by more than 2^8.  The weights
//            enter PV as two parts, so that they are not rounded to the
//            cache's type (one part: 1.4 times the output error).
//
// F32: x = hi + lo in fp16, hi x rounded and lo the rest: 22 bits of every
// element above 2^-17 of the largest that shares its scale.  A query row has a
// scale of its own; the rows of a tile that a loader warp splits at a time share
// a power of two that puts their largest |x| in [2^14, 2^15); K's goes into the scores' factor, V's exponent e into the
// weights' exponent: p' = 2^(x + e - m), v' = v 2^-e, so that p' keeps its
// precision whatever the values' range, and l takes p' 2^-e.  m is an integer:
// x + (e - m) then rounds once, at the size of the exponent that matters.
//
// The tensor cores cut every addition to an accumulator off towards zero.  In S
// the small products go first, while the sum is small.  (High parts on one grid,
// whose products add up exactly, took the output error at head_dim 256 from 1.3
// to 0.8e-6 of the whole, but left an element 2^-12 of the largest only 11 bits:
// 2e-4 behind keys 2^10 times larger.)  O, 12 additions a tile, came out 1e-5 too
// small after 64 tiles of a stream: F32 adds it to a sum in global memory,
// rounded to nearest, every kFlush tiles and starts it again from zero.
//
// What bounds it (B200; bytes and products that it cannot do without against the
// measured 6540 GB/s and 1637 TFLOP/s; a pass from a graph, caches warm):
//   64 sequences, 16384 + 0..1000 bf16 rows, 28 heads on 4 of 128: 53 us; the
//     memory floor is 15 us, the tensor floor (three products' time for two)
//     14; nothing is full (tensor pipe 45 %, issue slots 25 %, DRAM 25 %, L2
//     19 %): a tile takes its CTA 0.9 us, a chain of scores, maximum, exponentials,
//     parts and hand-over that the two streams overlap only in part, and the ends
//     of some 400 segments cost 3 us each;
//   16 sequences, 4093 + 1..700 F32 rows: 31 us, floor 6; one tile takes its
//     CTA 2 us, most of it in the loaders' splitting and the softmax's waits
//     (tensor pipe 17 %, DRAM 18 %, instruction cache hits 81 %);
//   5 sequences, 333 + 100..2000 F32 rows at head_dim 256: 46 us, floor 7; one
//     softmax stream for half of the value columns, 64 KB of keys split for each,
//     and 8 us a segment to bring Q's two parts into TMEM;
//   8 sequences, 3001..8191 f16 rows, 16 heads on 8 of 64: 39 us, floor 14; the
//     same chain, of which 2 of 32 lanes hold a query row;
//   one sequence of 812 F32 rows: 17 us, of which each CTA's single tile takes 8
//     from launch to partial, all latency: lengths, Q, rows, S, weights, PV in turn.
//
// TMEM columns: S/P buffers from 0, then Q, O up to 511.  Every wait is bounded.
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "lalb_batch.cuh"
#include "lalb_tcgen05.cuh"

using namespace lalb;

namespace {

constexpr int kGrid = 148;           // one CTA per SM of a B200 (workspace sizes need no device)
constexpr int kTile = 64;            // cache rows per tile
constexpr int kM = 128;              // query rows per unit
constexpr int kFew = 16;             // units of at most so many rows: a tile's columns are split over the warps
// list places a unit takes beside its tiles: what its segment's ends cost
constexpr int kPad16 = 3, kPadF32 = 2;
constexpr int kLens = 512;           // sequences whose lengths a CTA keeps in shared memory
constexpr int kSide = 8;             // tiles whose F32 scales are kept (Cfg checks that they outlive the ring)
// F32: a stream's tiles between two additions of its O to the sum in memory (1, 2,
// 4: 39, 36, 31 us for 16 sequences behind 4093 rows, and output errors of 0.6,
// 0.7 and 0.9e-6 of the whole)
constexpr int kFlush = 4;
constexpr float kShift = 6.0f;       // weights up to 2^6 at the reference maximum, 2^14 before a rescale
constexpr float kGrow = 8.0f;        // growth of a row's maximum that is left in place
constexpr int kStageBudget2 = 160 * 1024, kStageBudget1 = 192 * 1024, kStageBudgetRaw = 128 * 1024;

template <class T, int HD>
struct Cfg {
    static constexpr bool kF32 = sizeof(T) == 4;
    using H = typename std::conditional<kF32, __half, T>::type;   // the operands' type
    // F32 at head_dim 256: Q's two parts take 256 TMEM columns, so a unit has
    // half of the value columns (the scores are computed for both halves)
    static constexpr int kDV = kF32 && HD == 256 ? 128 : HD;
    static constexpr int kNDV = HD / kDV;
    static constexpr int kQCols = kF32 ? HD : HD / 2;
    static constexpr int kNS = 2 * kTile + kQCols + 2 * kDV <= 512 ? 2 : 1;   // softmax streams
    // score buffers: S runs kBufs - 1 tiles ahead of PV.  With two streams and
    // one tile ahead a stream's next scores wait behind its own last product
    // (2.1 us for a pair of tiles whose products take 0.8); a third buffer
    // needs 64 columns that F32 at head_dim 128 does not have
    static constexpr int kBufs = kNS == 2 && 3 * kTile + kQCols + 2 * kDV <= 512 ? 3 : 2;
    static constexpr int kAhead = kBufs - 1;
    static constexpr int kColS = 0, kColQ = kBufs * kTile, kColO = 512 - kNS * kDV;
    static_assert(kColQ + kQCols <= kColO, "the buffers, Q and O fit TMEM");
    static constexpr int kSoftWarps = 4 * kNS;
    // F32: 7, which with the MMA warp makes two warpgroups
    static constexpr int kLoadWarps = kF32 ? 7 : 1;
    // F32: rows that a loader warp splits at a time, under one power of two
    static constexpr int kRows = HD == 256 ? 8 : 16, kGroups = kTile / kRows;
    static constexpr int kFullCount = kF32 ? kGroups : 1;    // arrivals that fill a stage
    static constexpr int kOtherWarps = kF32 ? 8 : 4;   // MMA, loaders (16 bits: two warps idle)
    static constexpr int kThreads = 32 * (kSoftWarps + kOtherWarps);
    // Registers a thread: the launch's even share, and the split of it (the
    // softmax holds a tile's scores and weights; at the even share it spills)
    static constexpr int kEven = kThreads == 512 ? 128 : kThreads == 384 ? 168 : 248;
    static constexpr int kSoftRegs = kF32 ? (kNS == 2 ? 152 : 232) : kNS == 2 ? 200 : 0;   // 0: no split
    static constexpr int kOtherRegs = kF32 ? (kNS == 2 ? 104 : 136) : 104;
    static_assert(kSoftRegs == 0 || kSoftRegs * kSoftWarps + kOtherRegs * kOtherWarps <=
                                        kEven * (kSoftWarps + kOtherWarps),
                  "the split is no more than the block was launched with");
    static constexpr uint32_t kStage = kTile * HD * (kF32 ? 4 : 2);
    // F32 rows come in raw, a group at a time, into a slot of the loader warp
    // that splits them (head_dim 256 has no room: plain loads)
    static constexpr bool kRaw = kF32 && kDV == HD;
    static constexpr uint32_t kGroup = kRows * HD * 4;
    static constexpr int kSlots = HD == 128 ? 1 : 2;
    static constexpr int kBudget = kRaw ? kStageBudgetRaw : kNS == 2 ? kStageBudget2 : kStageBudget1;
    // F32 at head_dim 256: two slots of K (64 KB) and two of V's half (32) instead of
    // three of 64, in which a tile's K had to wait for the V two tiles before (4.5
    // us a tile)
    static constexpr bool kTwoRings = kNDV == 2;
    static constexpr int kStages = kTwoRings ? 4 : kBudget / (int)kStage < 10 ? kBudget / (int)kStage : 10;
    static_assert(kStages >= 2 * kAhead + 1, "V(j) to K(j + kAhead) are held at once");
    // Stage st = 2 t (K of the CTA's tile t) or 2 t + 1 (its V): its slot, how often
    // the slot was used before, and the slot's place
    static __device__ __forceinline__ uint32_t slot(uint32_t st) {
        return kTwoRings ? 2 * (st & 1) + (st >> 1 & 1) : st % kStages;
    }
    static __device__ __forceinline__ uint32_t uses(uint32_t st) { return kTwoRings ? st >> 2 : st / kStages; }
    static __device__ __forceinline__ uint32_t place(uint32_t slot) {
        return kTwoRings && slot >= 2 ? 2 * kStage + (slot - 2) * (kStage / 2) : slot * kStage;
    }
    static_assert(kStages / 2 + 2 <= kSide, "a tile's scales outlive its stages");
    // Narrow heads' tiles come in faster than one warp weighs them (8 sequences
    // of 3001 to 8191 scored f16 rows at head_dim 64: 45 us without, 39 with; F32
    // 70 and 69); wide ones wait for memory or the loaders, and four Qs and the
    // sum at the end cost more than they give (64 sequences of up to 1000 bf16
    // rows behind a prefix, head_dim 128: 69 and 77; one of 64 F32 rows 17 and 18)
    static constexpr bool kFewOk = HD <= 64;
    static constexpr int kSubW = HD < 64 ? HD : 64;                   // columns of a swizzled subtile
    static constexpr uint32_t kSub = kTile * kSubW * 2;               // its bytes
    static constexpr uint32_t kOffScratch = kTwoRings ? 3 * kStage : kStages * kStage;   // 4 KB per softmax warp
    static constexpr uint32_t kOffRaw = kOffScratch + kSoftWarps * 4096;
    static constexpr uint32_t kOffMl = kOffRaw + (kRaw ? kLoadWarps * kSlots * kGroup : 0);
    // (m, l) and, F32, each query row's largest |q|: per stream and row, of two segments
    static constexpr uint32_t kOffSide = kOffMl + 2 * 2 * kM * (kF32 ? 12 : 8);
    static constexpr uint32_t kOffLens = kOffSide + kSide * 16 * 4;
    static constexpr uint32_t kOffBar = kOffLens + kLens * 4;
    static constexpr uint32_t kSmem = 1024 + kOffBar + 512;
    static_assert(kSmem <= 232448, "fits the 227 KB opt-in shared memory");
    static_assert(kSmem > 116 * 1024 || kStages == 10, "one CTA per SM is what the ring is sized for");
};

struct AbArgs {
    const void *q, *pk, *pv, *k, *v;   // pk .. v: F32 loaders only
    const int *lens;
    int *cum;                    // [n_seq + 1] list places of the sequences before b (one unit each)
    float *part_p, *part_o;      // partial O of prefix and own units
    float2 *ml_p, *ml_o;         // their (m, l)
    float *sum;                  // F32: [CTA][stream][value column][row] O of the segment's earlier tiles
    float *score;                // add_weights: x_j [n_seq][n_head][pitch]
    float *row_weight;
    void *out;
    unsigned int *status;
    long long q_stride;
    int n_seq, n_head, n_kv, group, max_ctx, prefix, add_weights;
    int m_p, m_o;                // 128-row tiles of a prefix and an own unit's KV head
    int rows_p, rows_o;          // rows kept per partial: query rows of a prefix and an own unit at most
    int pitch, pad;              // score rows' distance; empty list places of a unit
    float c, decay, sign;        // |scale| log2 e, sign of the scale
};

__host__ __device__ inline int tiles_of(int rows) { return (rows + kTile - 1) / kTile; }

// List places of a unit over n rows: its tiles after `pad` empty ones.
__host__ __device__ inline int places_of(int rows, int pad) { return rows > 0 ? pad + tiles_of(rows) : 0; }

// A length outside the cache counts as 0.
__device__ __forceinline__ int checked_len(const AbArgs &a, int n) { return n < 0 || n > a.max_ctx ? 0 : n; }

// The list: the prefix units' places first, then per sequence its units'.
// CTA c takes `per` places, the first `rem` CTAs one more.  A segment's ends
// (Q, the pipeline's fill and drain, the partial) take as long as two or three
// tiles; without empty places for them, CTAs with many short units finish last
// (64 sequences of up to 1000 rows behind a prefix of 16384, bf16: 69 us, with
// 3 places 52, with 2 or 4 60 and 54; 30 F32 sequences of up to 1000 rows: 43, 41
// and 46 with 3, 2 and 4, 50 of up to 100 behind 1000: 35 and 31 with 3 and 2).
// (The host bounds every index.)
struct List {
    int tp, total;         // places of the prefix units, all places
    int lt;                // places of a prefix unit
    int units_o;           // own units per sequence
    int per, rem;

    __device__ __forceinline__ List(const AbArgs &a, int ndv, int own_places) {
        lt = places_of(a.prefix, a.pad);
        tp = a.n_kv * a.m_p * ndv * lt;
        units_o = a.n_kv * a.m_o * ndv;
        total = tp + own_places * units_o;
        per = total / kGrid;
        rem = total - per * kGrid;
    }
    __device__ __forceinline__ int first(int c) const { return c * per + min(c, rem); }
    __device__ __forceinline__ int owner(int t) const {
        const int big = (per + 1) * rem;
        return t < big ? t / (per + 1) : rem + (t - big) / per;
    }
};

struct Seg {
    bool prefix;
    int b;                 // own units: the sequence
    int g, m, dv;
    int j0, j1;            // tiles of the unit
    int n;                 // rows of the unit's cache
    int rows;              // query rows of the unit
    int slot;              // partial
};

// Walks one CTA's segments.  Every role walks on its own.
struct Walk {
    int t, end;
    int b;
    int c0;                // list place of sequence b's first, less tp
    int n, np;             // length and places of a unit of sequence b
    const int *lens_s;     // the first kLens lengths

    template <int NDV>
    __device__ __forceinline__ bool next(const AbArgs &a, const List &l, Seg &s) {
#pragma unroll 1
        for (;;) {
            if (t >= end) return false;
            int u, units, p0, places;
            if (t < l.tp) {
                u = t / l.lt;
                p0 = t - u * l.lt;
                places = l.lt;
                s.prefix = true;
                s.n = a.prefix;
                s.slot = blockIdx.x + u;
                units = a.m_p;
                s.b = 0;
            } else {
                const int o = t - l.tp;
#pragma unroll 1
                while (o >= c0 + np * l.units_o) {
                    c0 += np * l.units_o;
                    ++b;
                    n = checked_len(a, b < kLens ? lens_s[b] : __ldcg(a.lens + b));
                    np = places_of(n, a.pad);
                }
                u = (o - c0) / np;
                p0 = o - c0 - u * np;
                places = np;
                s.prefix = false;
                s.n = n;
                s.slot = blockIdx.x + b * l.units_o + u;
                units = a.m_o;
                s.b = b;
            }
            const int p1 = min(places, p0 + (end - t));
            t += p1 - p0;
            s.j0 = max(0, p0 - a.pad);
            s.j1 = p1 - a.pad;
            if (s.j1 <= s.j0) continue;      // empty places only
            const int v = u / NDV;
            s.dv = u - v * NDV;
            s.g = units == 1 ? v : v / units;
            s.m = v - s.g * units;
            s.rows = min(kM, (s.prefix ? a.n_seq * a.group : a.group) - s.m * kM);
            return true;
        }
    }
};

// ---- small PTX helpers -----------------------------------------------------------
// mbar_wait_bounded and warp_wait_fast with the retry loop kept rolled: the
// compiler unrolls its constant count at each of some twenty places, 55 KB of
// code in a kernel whose warps each run most of their path once or a few times
// and then wait for instructions.
__device__ __forceinline__ bool wait_bounded(uint64_t *bar, uint32_t parity, unsigned int *status) {
    if (mbar_test_wait(bar, parity)) return true;
#pragma unroll 1
    for (uint32_t i = 0; i < LALB_SPIN_LIMIT; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    atomicOr(status, LALB_STATUS_WAIT_TIMEOUT);
    return false;
}
// Every lane of the warp, which goes on only when all of them saw the phase complete.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, unsigned int *status) {
    return __all_sync(0xffffffffu, wait_bounded(bar, parity, status));
}

// 2^x within 2^-22 of it, 0 below 2^-126.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// A warpgroup's registers from here on (0: as launched).  In the role's own
// branch: where roles meet again the compiler keeps to the smaller share.
template <int N, bool INC>
__device__ __forceinline__ void set_regs() {
    if constexpr (N != 0 && INC)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N) : "memory");
    else if constexpr (N != 0)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N) : "memory");
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// x0, x1 as two 16-bit parts each: returns the pair of high parts, lo the
// rest.  Both are rounded to nearest, so that the two are within 2^-22 (fp16) or
// 2^-18 (bf16) of x, and the rests have either sign: F32's product of two
// rests, which is left out, is 0 on average and not 2^-22 of the whole.
template <class H>
__device__ __forceinline__ uint32_t split2(float2 x, uint32_t &lo) {
    const uint32_t hi = pack2<H>(x.x, x.y);
    float2 h;
    if constexpr (std::is_same<H, __half>::value)
        h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    else
        h = make_float2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u));
    const float2 r = __fadd2_rn(x, make_float2(-h.x, -h.y));
    lo = pack2<H>(r.x, r.y);
    return hi;
}

// Exponent e, 2^e the power of two that v 2^-e puts |v| <= amax below 2^15
// (and amax at or above 2^14), held in a range where 2^e and 2^-e stay normal.
__device__ __forceinline__ int part_exponent(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 127 - 14;
    return min(max(e, -74), 113);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// K-major tile (rows = tile rows, swizzled rows of kSubW 16-bit columns).
template <int SUBW>
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t saddr) {
    constexpr uint64_t sbo = SUBW * 2 * 8, type = SUBW == 64 ? 2 : 4;
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((sbo >> 4) << 32) | ((uint64_t)1 << 46) |
           (type << 61);
}
// The same bytes read along the rows: columns are N, tile rows are K.  The
// next 64 columns are one subtile on, the next 8 rows one swizzle atom.
template <int SUBW>
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t saddr) {
    constexpr uint64_t sbo = SUBW * 2 * 8, type = SUBW == 64 ? 2 : 4, lbo = kTile * SUBW * 2;
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((lbo >> 4) << 16) | ((sbo >> 4) << 32) | ((uint64_t)1 << 46) |
           (type << 61);
}

template <class T>
constexpr uint32_t mma_idesc(int n, bool b_mn) {
    const uint32_t t = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;   // bf16 : fp16
    return (1u << 4) | (t << 7) | (t << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kM >> 4) << 24);
}

// ---- F32 loaders: a group of ROWS rows of a tile by one warp ----------------------------
// COLS columns of each (rows at or past the end are zeros): registers first,
// then split and stored.
template <int COLS, int ROWS>
struct RowLoad {
    static constexpr int kLanes = COLS / 4 < 32 ? COLS / 4 : 32;   // lanes of one row
    static constexpr int kPer = 32 / kLanes;                       // rows per load
    static constexpr int kVec = COLS / (4 * kLanes);               // loads of one row
    static constexpr int kN = ROWS / kPer * kVec;
    float4 x[kN];

    __device__ __forceinline__ void load(const float *src, size_t pitch, int left, int lane) {
        const int rr = lane / kLanes, cc = (lane % kLanes) * 4;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int r = i / kVec * kPer + rr, c = cc + (i % kVec) * 4 * kLanes;
            x[i] = r < left ? __ldg(reinterpret_cast<const float4 *>(src + (size_t)r * pitch + c))
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    // The same from the rows as they lie in shared memory.
    __device__ __forceinline__ void load_raw(const uint8_t *raw, int left, int lane) {
        const int rr = lane / kLanes, cc = (lane % kLanes) * 4;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int r = i / kVec * kPer + rr, c = cc + (i % kVec) * 4 * kLanes;
            x[i] = r < left ? *reinterpret_cast<const float4 *>(raw + r * (COLS * 4) + c * 4)
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    // The rows' common exponent: that of their largest finite |x|, so that an
    // infinity spoils its own products only.  2 x bits + 2^24 drops the sign, and
    // infinities and NaNs wrap around to less than any other value.
    __device__ __forceinline__ int exponent() const {
        uint32_t m4[4] = {0, 0, 0, 0};
        auto key = [](float v) { return 2 * __float_as_uint(v) + (1u << 24); };
#pragma unroll
        for (int i = 0; i < kN; ++i)
            m4[i & 3] = max(m4[i & 3], max(max(key(x[i].x), key(x[i].y)), max(key(x[i].z), key(x[i].w))));
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(max(m4[0], m4[1]), max(m4[2], m4[3])));
        return part_exponent(__uint_as_float((max(m, 1u << 24) - (1u << 24)) >> 1));
    }
    __device__ __forceinline__ void store(uint8_t *stage, int r0, float scale, int lane) const {
        constexpr int W = COLS < 64 ? COLS : 64;
        constexpr uint32_t kLo = kTile * COLS * 2;
        const int rr = lane / kLanes, cc = (lane % kLanes) * 4;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int r = r0 + i / kVec * kPer + rr, c = cc + (i % kVec) * 4 * kLanes;
            uint2 hi, lo;
            const float2 a = make_float2(x[i].x * scale, x[i].y * scale), b = make_float2(x[i].z * scale, x[i].w * scale);
            hi.x = split2<__half>(a, lo.x);
            hi.y = split2<__half>(b, lo.y);
            const int unit = (c % W) >> 3;
            const int sw = W == 64 ? unit ^ (r & 7) : unit ^ ((r >> 1) & 3);
            const uint32_t off = (uint32_t)(c / W) * (kTile * W * 2) + r * (W * 2) + sw * 16 + (c & 4) * 2;
            *reinterpret_cast<uint2 *>(stage + off) = hi;
            *reinterpret_cast<uint2 *>(stage + off + kLo) = lo;
        }
    }
};

template <class T, int HD>
__global__ void __launch_bounds__(Cfg<T, HD>::kThreads, 1)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap mPK, const __grid_constant__ CUtensorMap mPV,
                           const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV,
                           const __grid_constant__ AbArgs a) {
    using C = Cfg<T, HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float *side = reinterpret_cast<float *>(smem + C::kOffSide);      // [tile % kSide][K 8, V 8]
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::kOffBar);
    uint64_t *empty = full + C::kStages;
    uint64_t *sfull = empty + C::kStages;      // S(j) complete (and every product issued before it)
    uint64_t *pready = sfull + C::kBufs;       // P(j) written
    uint64_t *ofull = pready + C::kBufs;       // a stream's latest PV complete
    uint64_t *qready = ofull + 2;              // Q of the segment written
    uint64_t *oready = qready + 1;             // O of the segment read
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(oready + 1);
    uint64_t *rawfull = reinterpret_cast<uint64_t *>(smem + C::kOffBar + 384);    // [loader warp][slot]
    int *start_b = reinterpret_cast<int *>(tmem_slot + 1);
    int *start = start_b + 1;                  // own tiles of all, of those before start_b, start_b's length

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], C::kFullCount);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < C::kBufs; ++s) {
            mbar_init(&sfull[s], 1);
            mbar_init(&pready[s], 4);
        }
        for (int s = 0; s < 2; ++s) mbar_init(&ofull[s], 1);
        if constexpr (C::kRaw)
            for (int k = 0; k < C::kSlots * C::kLoadWarps; ++k) mbar_init(&rawfull[k], 1);
        mbar_init(qready, C::kSoftWarps);
        mbar_init(oready, C::kSoftWarps);
        fence_barrier_init();
    }
    if (warp == C::kSoftWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    pdl_wait();
    // ---- the list: its length, and where this CTA's own tiles begin ---------------------
    // the lengths, one read for all of them
    int *lens_s = reinterpret_cast<int *>(smem + C::kOffLens);
    for (int b = threadIdx.x; b < a.n_seq && b < kLens; b += C::kThreads) lens_s[b] = __ldcg(a.lens + b);
    __syncthreads();
    if (warp == 0) {
        auto length = [&](int b) { return b >= a.n_seq ? 0 : b < kLens ? lens_s[b] : __ldcg(a.lens + b); };
        auto scan = [&](int x) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            return x;
        };
        int sum = 0;
#pragma unroll 1
        for (int b0 = 0; b0 < a.n_seq; b0 += 32) {
            const int n = length(b0 + lane), nt = places_of(checked_len(a, n), a.pad), incl = scan(nt);
            if (blockIdx.x == 0) {
                if (n < 0 || n > a.max_ctx) atomicOr(a.status, LALB_STATUS_BAD_POSITION);
                if (b0 + lane < a.n_seq) a.cum[b0 + lane] = sum + incl - nt;
            }
            sum += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (blockIdx.x == 0 && lane == 0) a.cum[a.n_seq] = sum;
        const List l(a, C::kNDV, sum);
        const int first = l.first(blockIdx.x) - l.tp;   // among the own tiles
        // the sequence of that tile (the first one, if the CTA begins in the prefix)
        const int want = first > 0 ? first / l.units_o : 0;
        int sb = 0, before = 0, n0 = length(0);
        if (first > 0 && first < sum * l.units_o) {     // cum[sb] <= want < cum[sb + 1]
            int run = 0;
#pragma unroll 1
            for (int b0 = 0; b0 < a.n_seq; b0 += 32) {
                const int n = length(b0 + lane), nt = places_of(checked_len(a, n), a.pad), incl = scan(nt);
                const uint32_t past = __ballot_sync(0xffffffffu, run + incl > want);
                if (past) {
                    const int i = __ffs(past) - 1;
                    sb = b0 + i;
                    before = run + __shfl_sync(0xffffffffu, incl - nt, i);
                    n0 = __shfl_sync(0xffffffffu, n, i);
                    break;
                }
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
        if (lane == 0) {
            *start_b = sb;
            start[0] = sum;
            start[1] = before;
            start[2] = checked_len(a, n0);
        }
    }
    __syncthreads();
    pdl_launch_dependents();   // after the allocation: a dependent that allocates TMEM too must not come first
    tc_after();
    const uint32_t tmem = *tmem_slot;
    // with the whole of TMEM allocated its base is column 0; anything else
    // raises a status bit and skips the work
    const bool tmem_ok = tmem == 0;
    if (!tmem_ok && threadIdx.x == 0) atomicOr(a.status, LALB_STATUS_WAIT_TIMEOUT);
    const List list(a, C::kNDV, start[0]);
    Walk walk;
    walk.t = list.first(blockIdx.x);
    walk.end = tmem_ok ? list.first(blockIdx.x + 1) : 0;
    walk.b = *start_b;
    walk.c0 = start[1] * list.units_o;
    walk.n = start[2];
    walk.np = places_of(walk.n, a.pad);
    walk.lens_s = lens_s;
    Seg s;

    if (warp > C::kSoftWarps + C::kLoadWarps) {
        set_regs<C::kSoftRegs ? C::kOtherRegs : 0, false>();     // idle
    } else if (warp > C::kSoftWarps) {
        set_regs<C::kSoftRegs ? C::kOtherRegs : 0, false>();
        // ================================ loaders ===============================================
        if constexpr (C::kF32) {
            // A stage is kGroups groups of rows, which go round the loader warps:
            // warp w has groups w, w + 7, w + 14, .. of the CTA's stages.
            const size_t pitch = (size_t)a.n_kv * HD;
            int k = warp - C::kSoftWarps - 1;            // the next group to look at
            int t0 = 0, t1 = 0;                          // the segment's tiles, counted over the CTA
            const float *kb = nullptr, *vb = nullptr;
            bool ok = true;
            struct Task {
                const float *p;      // plain loads: the rows
                int left, k;         // rows of the cache from the first one on; the group's number
                int row;             // raw: the first row in its tensor map
                bool prefix;
            };
            auto advance = [&](Task &t) -> bool {
                const int tile = k / (2 * C::kGroups);
#pragma unroll 1
                while (tile >= t1) {
                    if (!walk.template next<C::kNDV>(a, list, s)) return false;
                    t0 = t1;
                    t1 += s.j1 - s.j0;
                    const size_t seq = s.prefix ? 0 : (size_t)s.b * a.max_ctx * pitch;
                    kb = static_cast<const float *>(s.prefix ? a.pk : a.k) + seq + (size_t)s.g * HD;
                    vb = static_cast<const float *>(s.prefix ? a.pv : a.v) + seq + (size_t)s.g * HD + s.dv * C::kDV;
                }
                const int row = (s.j0 + tile - t0) * kTile + C::kRows * (k % C::kGroups);
                t.p = (k / C::kGroups & 1 ? vb : kb) + (size_t)row * pitch;
                t.left = s.n - row;
                t.row = row + (s.prefix ? 0 : s.b * a.max_ctx);
                t.prefix = s.prefix;
                t.k = k;
                k += C::kLoadWarps;
                return true;
            };
            auto finish = [&](const auto &x, int k, int e) {
                const uint32_t st = k / C::kGroups, g = k % C::kGroups, slot = C::slot(st), use = C::uses(st);
                if (use > 0) ok = ok && warp_wait(&empty[slot], (use - 1) & 1u, a.status);
                x.store(smem + C::place(slot), C::kRows * g, pow2(-e), lane);
                // K: the factor that undoes the scaling; V: the exponent
                if (lane == 0) side[((st >> 1) % kSide) * 16 + (st & 1) * 8 + g] = st & 1 ? (float)e : pow2(e);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[slot]);
            };
            Task t;
            if constexpr (C::kRaw) {
                // kSlots groups on their way: the next starts into a slot as soon as the
                // warp has its rows in registers
                const int w = warp - C::kSoftWarps - 1;
                uint8_t *raw = smem + C::kOffRaw + w * C::kSlots * C::kGroup;
                uint64_t *bar = rawfull + C::kSlots * w;
                auto issue = [&](const Task &u, int slot) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&bar[slot], C::kGroup);
                        const bool v = u.k / C::kGroups & 1;
                        const CUtensorMap *m = u.prefix ? (v ? &mPV : &mPK) : (v ? &mV : &mK);
                        tma2d(raw + slot * C::kGroup, m, s.g * HD, u.row, &bar[slot]);
                    }
                };
                Task q0, q1;
                int issued = 0, taken = 0;
                if (advance(q0)) issue(q0, 0), ++issued;
                if (C::kSlots == 2 && issued && advance(q1)) issue(q1, 1), ++issued;
#pragma unroll 1
                while (taken < issued && ok) {
                    const int slot = taken % C::kSlots;
                    const int left = slot ? q1.left : q0.left, kk = slot ? q1.k : q0.k;
                    ok = warp_wait(&bar[slot], (taken / C::kSlots) & 1u, a.status);
                    RowLoad<HD, C::kRows> x;
                    x.load_raw(raw + slot * C::kGroup, left, lane);
                    const int e = x.exponent();      // the warp's maximum: every lane has its rows
                    ++taken;
                    if (issued == taken + C::kSlots - 1 && advance(t)) {
                        issue(t, slot);
                        ++issued;
                        if (slot)
                            q1 = t;
                        else
                            q0 = t;
                    }
                    finish(x, kk, e);
                }
                // nothing may still be on its way into this CTA's shared memory when it ends
                for (; taken < issued; ++taken) (void)warp_wait(&bar[taken % C::kSlots], (taken / C::kSlots) & 1u, a.status);
            } else {
#pragma unroll 1
                while (ok && advance(t)) {
                    if (t.k / C::kGroups & 1) {
                        RowLoad<C::kDV, C::kRows> x;
                        x.load(t.p, pitch, t.left, lane);
                        finish(x, t.k, x.exponent());
                    } else {
                        RowLoad<HD, C::kRows> x;
                        x.load(t.p, pitch, t.left, lane);
                        finish(x, t.k, x.exponent());
                    }
                }
            }
        } else if (lane == 0) {
            uint32_t st = 0;
            bool ok = true;
#pragma unroll 1
            while (walk.template next<C::kNDV>(a, list, s)) {
                const CUtensorMap *mk = s.prefix ? &mPK : &mK, *mv = s.prefix ? &mPV : &mV;
                const int row0 = s.prefix ? 0 : s.b * a.max_ctx;
#pragma unroll 1
                for (int j = s.j0; j < s.j1 && ok; ++j)
#pragma unroll 1
                    for (int kv = 0; kv < 2 && ok; ++kv, ++st) {
                        const uint32_t slot = C::slot(st), use = C::uses(st);
                        if (use > 0 && !wait_bounded(&empty[slot], (use - 1) & 1u, a.status)) {
                            ok = false;
                            break;
                        }
                        mbar_arrive_expect_tx(&full[slot], C::kStage);
#pragma unroll
                        for (int c = 0; c < HD / C::kSubW; ++c)
                            tma2d(smem + C::place(slot) + c * C::kSub, kv ? mv : mk, s.g * HD + c * C::kSubW,
                                  row0 + j * kTile, &full[slot]);
                    }
            }
            // nothing may still be on its way into this CTA's shared memory when it ends
#pragma unroll 1
            for (uint32_t i = st > (uint32_t)C::kStages ? st - C::kStages : 0; i < st; ++i)
                wait_bounded(&full[C::slot(i)], C::uses(i) & 1u, a.status);
        }
    } else if (warp == C::kSoftWarps) {
        // ================================ MMA ====================================================
        set_regs<C::kSoftRegs ? C::kOtherRegs : 0, false>();
        constexpr uint32_t kIdS = mma_idesc<typename C::H>(kTile, false);
        constexpr uint32_t kIdO = mma_idesc<typename C::H>(C::kDV, true);
        constexpr uint32_t kLoK = kTile * HD * 2, kLoV = kTile * C::kDV * 2;
        const uint32_t ring = smem_u32(smem);
        uint32_t tile = 0, segs = 0;        // tiles before the segment: its K(i) is stage 2 (tile + i)
        bool ok = true;
        auto issue_pv = [&](uint32_t t, bool first) -> bool {
            const uint32_t buf = t % C::kBufs, sv = C::slot(2 * t + 1), use = C::uses(2 * t + 1);
            if (!warp_wait(&pready[buf], (t / C::kBufs) & 1u, a.status) ||
                !warp_wait(&full[sv], use & 1u, a.status))
                return false;
            tc_after();
            const uint32_t stream = C::kNS == 2 ? t & 1u : 0;
            const uint32_t d = C::kColO + stream * C::kDV, p = C::kColS + buf * kTile, v = ring + C::place(sv);
            // weights: of 16 scores' 16 columns, 8 hold the high parts, 8 the rest
            auto hi = [&](int kk) { return p + 16 * kk; };
            auto v_off = [&](int kk) { return v + kk * 16 * C::kSubW * 2; };
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk) {
                if constexpr (C::kF32)
                    mma_f16_ta(d, hi(kk), mnmajor_desc<C::kSubW>(v_off(kk) + kLoV), kIdO, first && kk == 0 ? 0u : 1u);
                mma_f16_ta(d, hi(kk) + 8, mnmajor_desc<C::kSubW>(v_off(kk)), kIdO,
                           first && kk == 0 && !C::kF32 ? 0u : 1u);
            }
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
                mma_f16_ta(d, hi(kk), mnmajor_desc<C::kSubW>(v_off(kk)), kIdO, 1u);
            commit_elect(&empty[sv]);
            commit_elect(&ofull[stream]);
            return true;
        };
#pragma unroll 1
        while (ok && walk.template next<C::kNDV>(a, list, s)) {
            if (!(ok = warp_wait(qready, segs & 1u, a.status))) break;
            tc_after();
            ++segs;
            const int n = s.j1 - s.j0;
#pragma unroll 1
            for (int i = 0; i < n + C::kAhead && ok; ++i) {
                if (i < n) {
                    const uint32_t t = tile + i, buf = t % C::kBufs;
                    const uint32_t sk = C::slot(2 * t), use = C::uses(2 * t);
                    if (!(ok = warp_wait(&full[sk], use & 1u, a.status))) break;
                    tc_after();
                    const uint32_t d = C::kColS + buf * kTile, k = ring + C::place(sk);
                    auto k_off = [&](int kk) {
                        return k + (kk / (C::kSubW / 16)) * C::kSub + (kk % (C::kSubW / 16)) * 32;
                    };
                    // The tensor cores cut each sum off towards zero at its own size: the
                    // small products go first, while the sum is small.
                    if constexpr (C::kF32) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            mma_f16_ta(d, C::kColQ + 8 * kk, kmajor_desc<C::kSubW>(k_off(kk) + kLoK), kIdS, kk ? 1u : 0u);
                            mma_f16_ta(d, C::kColQ + HD / 2 + 8 * kk, kmajor_desc<C::kSubW>(k_off(kk)), kIdS, 1u);
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk)
                        mma_f16_ta(d, C::kColQ + 8 * kk, kmajor_desc<C::kSubW>(k_off(kk)), kIdS, kk || C::kF32 ? 1u : 0u);
                    commit_elect(&empty[sk]);
                    commit_elect(&sfull[buf]);
                }
                if (i >= C::kAhead) {
                    const int j = i - C::kAhead;
                    // the last segment's O is read by now, or will be soon
                    if (j == 0 && segs > 1 && !(ok = warp_wait(oready, segs & 1u, a.status))) break;
                    const int mine = j / C::kNS;       // the stream's tile of the segment
                    ok = issue_pv(tile + j, C::kF32 ? mine % kFlush == 0 : mine == 0);
                }
            }
            tile += n;
        }
    } else {
        // ================================ softmax ==================================================
        set_regs<C::kSoftRegs, true>();
        const int wg = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        uint8_t *scratch = smem + C::kOffScratch + warp * 4096;
        // Two of each, taken in turn: a warpgroup without a tile in a segment may
        // be at the next boundary while the other still reads this one's.
        float2 *ml = reinterpret_cast<float2 *>(smem + C::kOffMl);    // [stream][row]: (m, l)
        float *qmax = reinterpret_cast<float *>(ml + 2 * 2 * kM);     // F32: [warpgroup][row], largest |q| of its columns
        uint32_t turn = 0;
        uint32_t tile = 0;                      // before the segment
        uint32_t pv0 = 0, pv1 = 0;              // products of each stream so far
        bool ok = true;
        auto wg_bar = [&]() {      // one warpgroup
            if (C::kNS == 2 && wg)
                asm volatile("bar.sync 3, 128;" ::: "memory");
            else
                asm volatile("bar.sync 2, 128;" ::: "memory");
        };
        auto soft_bar = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(32 * C::kSoftWarps) : "memory"); };

        // ---- Q: this warp's 32 rows, the 32-column chunks of its warpgroup, into TMEM ----------------
        // Loaded kLpr lanes to a row (whole sectors), turned to a row per lane in
        // the warp's scratch memory.  A batch is what the registers hold.
        constexpr int kLpr = 2 * sizeof(T), kRpi = 32 / kLpr, kIt = 32 / kRpi;   // lanes per row, rows per load
        constexpr int kChunks = HD / 32 < C::kNS ? 1 : HD / 32 / C::kNS;        // of this warpgroup
        const bool q_idle = wg >= HD / 32;      // head_dim 32: one chunk, the first warpgroup's
        constexpr int kBatch = 16 / kIt < kChunks ? 16 / kIt : kChunks;         // chunks per batch
        const int lr = lane / kLpr, lu = lane % kLpr;
        auto few = [&](const Seg &g) { return C::kFewOk && (g.prefix ? a.rows_p : a.rows_o) <= kFew; };
        auto first_row = [&](const Seg &g) { return few(g) ? 0 : quarter * 32; };   // the warp's first row
        auto q_load = [&](const Seg &g, int c0, uint4 (&v)[kBatch * kIt]) {
            const T *qb = static_cast<const T *>(a.q) + (size_t)g.g * a.group * HD + (c0 * C::kNS + wg) * 32;
            // row r of the unit: head h of sequence b, and kRpi rows further each time
            int r = first_row(g) + lr, b = g.b, h = g.m * kM + r;
            if (g.prefix) {
                b = h / a.group;
                h -= b * a.group;
            }
#pragma unroll
            for (int i = 0; i < kIt; ++i) {
                const T *p = qb + (size_t)b * a.q_stride + (size_t)h * HD;
#pragma unroll
                for (int c = 0; c < kBatch; ++c)
                    v[c * kIt + i] = r < g.rows ? __ldg(reinterpret_cast<const uint4 *>(p + c * C::kNS * 32) + lu)
                                                : make_uint4(0, 0, 0, 0);
                r += kRpi;
                h += kRpi;
                if (g.prefix)
#pragma unroll 1
                    while (h >= a.group) h -= a.group, ++b;
            }
        };
        // F32: the largest |q| in a batch, this lane's columns of its kIt rows
        auto q_top = [&](const uint4 (&v)[kBatch * kIt], float (&top)[kIt]) {
#pragma unroll
            for (int i = 0; i < kBatch * kIt; ++i)
                top[i % kIt] =
                    fmaxf(top[i % kIt], fmaxf(fmaxf(fabsf(__uint_as_float(v[i].x)), fabsf(__uint_as_float(v[i].y))),
                                              fmaxf(fabsf(__uint_as_float(v[i].z)), fabsf(__uint_as_float(v[i].w)))));
        };
        auto q_store = [&](int c0, const uint4 (&v)[kBatch * kIt], float qs) {
#pragma unroll
            for (int c = 0; c < kBatch; ++c) {
#pragma unroll
                for (int i = 0; i < kIt; ++i) {
                    const int r = i * kRpi + lr;
                    *reinterpret_cast<uint4 *>(scratch + r * 128 + ((lu ^ (r & 7)) << 4)) = v[c * kIt + i];
                }
                __syncwarp();
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int u = 0; u < kLpr; ++u) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(scratch + lane * 128 + ((u ^ (lane & 7)) << 4));
                    if constexpr (C::kF32) {
                        const float2 a0 = make_float2(__uint_as_float(x.x) * qs, __uint_as_float(x.y) * qs);
                        const float2 a1 = make_float2(__uint_as_float(x.z) * qs, __uint_as_float(x.w) * qs);
                        hi[2 * u] = split2<__half>(a0, lo[2 * u]);
                        hi[2 * u + 1] = split2<__half>(a1, lo[2 * u + 1]);
                    } else {
                        // a negative scale turns the queries' signs
                        const uint32_t f = qs < 0.0f ? 0x80008000u : 0u;
                        hi[4 * u] = x.x ^ f, hi[4 * u + 1] = x.y ^ f, hi[4 * u + 2] = x.z ^ f, hi[4 * u + 3] = x.w ^ f;
                    }
                }
                const uint32_t col = lanes + C::kColQ + 16 * ((c0 + c) * C::kNS + wg);
                tmem_st16(col, hi);
                if constexpr (C::kF32) tmem_st16(col + HD / 2, lo);
                __syncwarp();
            }
        };
        uint4 qv[kBatch * kIt];
        // before the barrier both warpgroups pass at a segment's start ..
        auto q_begin = [&](const Seg &g) {
            if (first_row(g) >= g.rows || q_idle) return;
            q_load(g, 0, qv);
        };
        auto q_share = [&](const Seg &g) {
            if constexpr (C::kF32) {
                if (first_row(g) >= g.rows || q_idle) return;
                float top[kIt] = {};
                q_top(qv, top);
#pragma unroll 1
                for (int c = kBatch; c < kChunks; c += kBatch) {
                    uint4 v[kBatch * kIt];
                    q_load(g, c, v);
                    q_top(v, top);
                }
                // over the kLpr lanes of a row, as many as a lane has rows: at each
                // step a lane hands on one half of its rows and keeps the other, at
                // the end it has row kRpi * lu + lr
                static_assert(kLpr == kIt, "a lane ends with one row");
#pragma unroll
                for (int o = kLpr / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < o; ++i) {
                        const bool up = lu & o;
                        const float away = up ? top[i] : top[i + o];
                        top[i] = fmaxf(up ? top[i + o] : top[i], __shfl_xor_sync(0xffffffffu, away, o));
                    }
                qmax[(turn * 2 + wg) * kM + quarter * 32 + kRpi * lu + lr] = top[0];
            }
        };
        // .. and after it: Q written (F32: each row under its own power of two, so that
        // no row's size, not even an infinity, reaches the rows of other heads and
        // sequences), the row's score factor returned
        auto q_finish = [&](const Seg &g) -> float {
            float qs = a.sign, cq = a.c;
            if (first_row(g) < g.rows) {
                if constexpr (C::kF32) {
                    const float *qm = qmax + turn * 2 * kM + row;
                    const int e = part_exponent(C::kNS == 2 && HD > 32 ? fmaxf(qm[0], qm[kM]) : qm[0]);
                    qs = a.sign * pow2(-e);
                    cq = a.c * pow2(e);
                }
                if (!q_idle) q_store(0, qv, qs);
#pragma unroll 1
                for (int c = kBatch; c < kChunks; c += kBatch) {
                    uint4 v[kBatch * kIt];
                    q_load(g, c, v);
                    q_store(c, v, qs);
                }
                tmem_wait_st();
            }
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(qready);
            return cq;
        };

        // F32: a stream's O, which starts again from zero, added to its sum (the
        // first time: put there)
        float *sum = nullptr;
        float mref = 0.0f, msum = 0.0f;          // reference exponents of O and of the sum
        if constexpr (C::kF32) sum = a.sum + (size_t)blockIdx.x * C::kNS * C::kDV * kM + row;
        auto flush = [&](uint32_t stream, bool first) {
            const float f = ex2(msum - mref);
            float *p = sum + stream * C::kDV * kM;
            constexpr int kC = C::kDV < 64 ? C::kDV : 64;    // columns whose sums are loaded together
#pragma unroll 1
            for (int c0 = 0; c0 < C::kDV; c0 += kC, p += kC * kM) {
                float v[kC];
#pragma unroll
                for (int k = 0; k < kC; ++k) v[k] = first ? 0.0f : p[k * kM];
#pragma unroll
                for (int c = 0; c < kC; c += 16) {
                    float o[16];
                    tmem_ld16_nowait(lanes + C::kColO + stream * C::kDV + c0 + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) p[(c + k) * kM] = first ? o[k] : fmaf(v[c + k], f, o[k]);
                }
            }
            msum = mref;
        };

        Seg nx;
        int n = 0;                               // the segment's tiles
        bool have = false, had = false;          // a segment is open; one of its tiles was this warpgroup's
        bool active = false;                     // a row of this warp belongs to its unit
        bool split = false;                      // at most 16 rows: this warp has 16 columns of a tile
        bool any = false;                        // this thread's row has met a score
        float cq = 0.0f, l = 0.0f;
#pragma unroll 1
        for (;;) {
            // ---- from one segment to the next ------------------------------------------------------
            // The next segment's Q is on its way while the last products run.  Each
            // warpgroup waits for its own stream's last one; past the barrier every
            // product is complete, Q and the score buffers are free, and the next
            // scores can start while O is read.
            const bool nhave = walk.template next<C::kNDV>(a, list, nx);
            if (nhave) q_begin(nx);
            // tiles of each stream in the segment
            const int cnt0 = C::kNS == 1 ? n : (n + 1 - (int)(tile & 1u)) / 2, cnt1 = n - cnt0;
            if (had) {
                const uint32_t k = C::kNS == 2 ? wg : 0;
                ok = ok && warp_wait(&ofull[k], ((k ? pv1 : pv0) - 1) & 1u, a.status);
                if constexpr (C::kF32) {
                    tc_after();
                    if (active && (k ? cnt1 : cnt0) > kFlush) flush(k, false);
                }
            }
            // (l is NaN where a score was, and says so even if all of them were)
            ml[turn * 2 * kM + wg * kM + row] = make_float2(had && (any || l != l) ? mref : -INFINITY, l);
            if (nhave) q_share(nx);
            tc_before();
            soft_bar();
            tc_after();
            const float2 *mlt = ml + turn * 2 * kM;
            const float2 r0 = mlt[row], r1 = C::kNS == 2 ? mlt[kM + row] : make_float2(-INFINITY, 0.0f);
            float cn = 0.0f;
            if (nhave) cn = q_finish(nx);
            turn ^= 1;
            if (have) {
                // a stream without a tile in this segment, or a score in this row, has nothing
                const bool has0 = r0.x > -INFINITY, has1 = r1.x > -INFINITY;
                float m = fmaxf(r0.x, r1.x), lsum = 0.0f;
                if (split) {       // the row's sums are in four warps
#pragma unroll
                    for (int k = 0; k < 4 * C::kNS; ++k) m = fmaxf(m, mlt[32 * k + lane].x);
#pragma unroll
                    for (int k = 0; k < 4 * C::kNS; ++k) {
                        const float2 x = mlt[32 * k + lane];
                        lsum = fmaf(x.y, x.x > -INFINITY ? ex2(x.x - m) : 0.0f, lsum);
                    }
                }
                const float f0 = has0 ? ex2(r0.x - m) : 0.0f, f1 = has1 ? ex2(r1.x - m) : 0.0f;
                if (active && (ok || split)) {     // split: all four warps meet at the barriers below
                    const int rows = s.prefix ? a.rows_p : a.rows_o;
                    const size_t first = (size_t)s.slot * rows + first_row(s);
                    float *po = (s.prefix ? a.part_p : a.part_o) + first * C::kDV;
                    float2 *pm = (s.prefix ? a.ml_p : a.ml_o) + first;
                    const int live = min(32, s.rows - first_row(s));
                    if (wg == 0 && lane < live && (!split || quarter == 0))
                        pm[lane] = make_float2(
                            m, split ? lsum : (has0 ? r0.y * f0 : 0.0f) + (has1 ? r1.y * f1 : 0.0f));
                    constexpr int kHalf = C::kDV / C::kNS, kP = 16;
                    constexpr int kOl = kP / 4, kOr = 32 / kOl;      // lanes of a row's piece, rows per store
                    const int olr = lane / kOl, olu = lane % kOl;
#pragma unroll 1
                    for (int c = wg * kHalf; c < (wg + 1) * kHalf; c += kP) {
                        float o[kP], v[kP];
                        tmem_ld16_nowait(lanes + C::kColO + c, o);
                        if constexpr (C::kNS == 2) tmem_ld16_nowait(lanes + C::kColO + C::kDV + c, v);
                        tmem_wait_ld();
                        if constexpr (C::kF32) {       // a stream with more tiles: its sum
                            if (cnt0 > kFlush) {
#pragma unroll
                                for (int k = 0; k < kP; ++k) o[k] = __ldcg(sum + (c + k) * kM);
                            }
                            if (C::kNS == 2 && cnt1 > kFlush) {
#pragma unroll
                                for (int k = 0; k < kP; ++k) v[k] = __ldcg(sum + (C::kDV + c + k) * kM);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < kP; ++k) {
                            o[k] = has0 ? o[k] * f0 : 0.0f;
                            if (C::kNS == 2 && has1) o[k] = fmaf(v[k], f1, o[k]);
                        }
                        if (split) {
                            // 64 columns of the warpgroup's at a time: each warp's rows side by
                            // side, then every thread adds the four warps' for its columns
                            constexpr int kW = kHalf < 64 ? kHalf : 64;
                            if (lane < live) {
#pragma unroll
                                for (int u = 0; u < kOl; ++u)
                                    *reinterpret_cast<float4 *>(scratch + lane * kW * 4 +
                                                                (((c % kW) / 4 + u) ^ (lane & (kW / 4 - 1))) * 16) =
                                        make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                            }
                            if ((c + kP) % kW) continue;
                            wg_bar();
                            const uint8_t *four = smem + C::kOffScratch + wg * 4 * 4096;
                            for (int i = quarter * 32 + lane; i < live * (kW / 4); i += 128) {
                                const int r = i / (kW / 4), u = i % (kW / 4);
                                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    const float4 v = *reinterpret_cast<const float4 *>(
                                        four + w * 4096 + r * kW * 4 + (u ^ (r & (kW / 4 - 1))) * 16);
                                    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                                }
                                *reinterpret_cast<float4 *>(po + (size_t)r * C::kDV + (c + kP - kW) + 4 * u) = sum;
                            }
                            wg_bar();
                            continue;
                        }
                        if (live <= 8) {      // a few rows: each lane its own
                            if (lane < live) {
#pragma unroll
                                for (int u = 0; u < kOl; ++u)
                                    *reinterpret_cast<float4 *>(po + (size_t)lane * C::kDV + c + 4 * u) =
                                        make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                            }
                            continue;
                        }
#pragma unroll
                        for (int u = 0; u < kOl; ++u)
                            *reinterpret_cast<float4 *>(scratch + lane * 128 + ((u ^ (lane & 7)) << 4)) =
                                make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                        __syncwarp();
#pragma unroll
                        for (int r = 0; r < 32; r += kOr)
                            if (r + olr < live)
                                *reinterpret_cast<float4 *>(po + (size_t)(r + olr) * C::kDV + c + 4 * olu) =
                                    *reinterpret_cast<const float4 *>(scratch + (r + olr) * 128 +
                                                                      ((olu ^ ((r + olr) & 7)) << 4));
                        __syncwarp();
                    }
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(oready);
                tile += n;
            }
            if (!nhave) break;
            // ---- this warpgroup's tiles ----------------------------------------------------------
            s = nx;
            have = true;
            cq = cn;
            n = s.j1 - s.j0;
            split = few(s);
            active = first_row(s) < s.rows;
            mref = l = 0.0f;
            any = false;
            had = false;
            float *score = nullptr;
            if (a.add_weights && !s.prefix && s.dv == 0 && first_row(s) + lane < s.rows)
                score = a.score +
                        ((size_t)s.b * a.n_head + (size_t)s.g * a.group + s.m * kM + first_row(s) + lane) * a.pitch;
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const uint32_t t = tile + i, buf = t % C::kBufs;
                const uint32_t stream = C::kNS == 2 ? t & 1u : 0;
                const uint32_t sv = 2 * t + 1;                  // the stage of the tile's values
                if (C::kNS == 1 || (int)stream == wg) {
                    // This stream's last product complete.  Every product is waited
                    // for, before the weights of the next are handed over, so that
                    // the barrier is never two phases away from a wait, where its
                    // parity would mislead.
                    const uint32_t done = stream ? pv1 : pv0;
                    bool waited = done == 0;
                    auto wait_pv = [&]() {
                        if (waited) return;
                        ok = ok && warp_wait(&ofull[stream], (done - 1) & 1u, a.status);
                        waited = true;
                        tc_after();
                    };
                    had = true;
                    const int valid = s.n - (s.j0 + i) * kTile;     // of the tile's 64 rows
                    ok = ok && warp_wait(&sfull[buf], (t / C::kBufs) & 1u, a.status);
                    tc_after();
                    if constexpr (C::kF32) {
                        const int k = i / C::kNS;       // the stream's tile of the segment
                        if (k > 0 && k % kFlush == 0) {
                            wait_pv();
                            if (active) flush(stream, k == kFlush);
                        }
                    }
                    if constexpr (!C::kF32) {
                        // stale rows behind a sequence's end may hold anything, NaN too,
                        // and 0 x NaN is NaN: the values' tile gets zeros there
                        if (!s.prefix && valid < kTile) {
                            ok = ok && warp_wait(&full[C::slot(sv)], C::uses(sv) & 1u, a.status);
                            uint8_t *v = smem + C::place(C::slot(sv));
                            constexpr int kU = C::kSubW * 2 / 16;
                            const int units = (kTile - valid) * kU;
#pragma unroll
                            for (int c = 0; c < HD / C::kSubW; ++c)
#pragma unroll 1
                                for (int u = quarter * 32 + lane; u < units; u += 128)
                                    *reinterpret_cast<uint4 *>(v + c * C::kSub + valid * C::kSubW * 2 + u * 16) =
                                        make_uint4(0, 0, 0, 0);
                            fence_async();
                        }
                    } else {
                        ok = ok && warp_wait(&full[C::slot(sv)], C::uses(sv) & 1u, a.status);
                    }
                    if (active && ok) {
                        const uint32_t sc = lanes + C::kColS + buf * kTile;
                        const float *sd = side + (t % kSide) * 16;
                        // never 0: -inf (a row past the end) times it has to stay -inf
                        auto factor = [&](int g) { return fmaxf(sd[8 * g / C::kRows] * cq, 1e-37f); };   // of columns 8 g ..
                        auto exponent = [&](int g) { return sd[8 + 8 * g / C::kRows]; };
                        auto past_end = [&](float *y, int j0, int nj) {
                            if (valid < kTile) {
#pragma unroll
                                for (int j = 0; j < nj; ++j)
                                    if (j0 + j >= valid) y[j] = -INFINITY;
                            }
                        };
                        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        // 16 bits: the tile's scores stay in registers.  F32: loops over 32
                        // or 16 of them, read again for the weights: unrolled, its longer
                        // code is fetched more slowly than the scores are read.
                        constexpr int kHeld = C::kF32 ? 1 : kTile;
                        float x[kHeld];
                        float few_x[16];
                        if (split) {
                            tmem_ld16_nowait(sc + 16 * quarter, few_x);
                            tmem_wait_ld();
                            past_end(few_x, 16 * quarter, 16);
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                const float f = C::kF32 ? factor(2 * quarter + g) : cq;
                                const float e = C::kF32 ? exponent(2 * quarter + g) : 0.0f;
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    top4[j & 3] = fmaxf(top4[j & 3], C::kF32 ? fmaf(few_x[8 * g + j], f, e)
                                                                             : few_x[8 * g + j]);
                                if (score) {
                                    float4 *o = reinterpret_cast<float4 *>(score + (s.j0 + i) * kTile + 16 * quarter);
#pragma unroll
                                    for (int j = 8 * g; j < 8 * g + 8; j += 4)
                                        o[j >> 2] = make_float4(few_x[j] * f, few_x[j + 1] * f, few_x[j + 2] * f,
                                                                few_x[j + 3] * f);
                                }
                            }
                        } else if constexpr (!C::kF32) {
                            tmem_ld32_nowait(sc, x);
                            tmem_ld32_nowait(sc + 32, x + 32);
                            tmem_wait_ld();
                            past_end(x, 0, kTile);
#pragma unroll
                            for (int j = 0; j < kTile; j += 8)
#pragma unroll
                                for (int q = 0; q < 4; ++q) top4[q] = fmaxf(top4[q], fmaxf(x[j + q], x[j + 4 + q]));
                            if (score) {
                                float4 *o = reinterpret_cast<float4 *>(score + (s.j0 + i) * kTile);
#pragma unroll
                                for (int j = 0; j < kTile; j += 4)
                                    o[j >> 2] = make_float4(x[j] * cq, x[j + 1] * cq, x[j + 2] * cq, x[j + 3] * cq);
                            }
                        } else {
#pragma unroll 1
                            for (int h = 0; h < 2; ++h) {
                                float y[32];
                                tmem_ld32_nowait(sc + 32 * h, y);
                                tmem_wait_ld();
                                past_end(y, 32 * h, 32);
#pragma unroll
                                for (int g = 0; g < 4; ++g) {
                                    const float f = factor(4 * h + g), e = exponent(4 * h + g);
#pragma unroll
                                    for (int j = 0; j < 8; j += 2) {
                                        const float2 v = __ffma2_rn(make_float2(y[8 * g + j], y[8 * g + j + 1]),
                                                                    make_float2(f, f), make_float2(e, e));
                                        top4[j >> 1] = fmaxf(top4[j >> 1], fmaxf(v.x, v.y));
                                    }
                                }
                                if (score) {
                                    float4 *o = reinterpret_cast<float4 *>(score + (s.j0 + i) * kTile + 32 * h);
#pragma unroll
                                    for (int j = 0; j < 32; j += 4) {
                                        const float f = factor(4 * h + (j >> 3));
                                        o[j >> 2] = make_float4(y[j] * f, y[j + 1] * f, y[j + 2] * f, y[j + 3] * f);
                                    }
                                }
                            }
                        }
                        float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
                        if constexpr (!C::kF32) top *= cq;
                        // ---- the reference exponent ----------------------------------------------------
                        // (a row with no score yet, all of them past the end, takes any: its l and O are 0)
                        const float want = top == -INFINITY ? mref : rintf(top) - kShift;
                        const bool grown = any && want > mref + kGrow;
                        if (!any) mref = want;
                        any = any || top > -INFINITY;
                        if (__any_sync(0xffffffffu, grown)) {
                            wait_pv();
                            const float to = grown ? want : mref;
                            const float f = ex2(mref - to);
                            mref = to;
                            l *= f;
                            const uint32_t oc = lanes + C::kColO + stream * C::kDV;
#pragma unroll 1
                            for (int c = 0; c < C::kDV; c += 16) {
                                float o[16];
                                tmem_ld16(oc + c, o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] *= f;
                                tmem_st16(oc + c, reinterpret_cast<const uint32_t *>(o));
                            }
                        }
                        // ---- weights -------------------------------------------------------------------
                        // 16 scores and their weights in their place: eight columns of high
                        // parts, eight of the rest
                        float2 sum2 = make_float2(0.0f, 0.0f);
                        auto weigh8 = [&](const float *y, float f, float e, uint32_t *hi, uint32_t *lo) {
#pragma unroll
                            for (int j = 0; j < 8; j += 2) {
                                const float2 v =
                                    __ffma2_rn(make_float2(y[j], y[j + 1]), make_float2(f, f), make_float2(e, e));
                                const float2 p = make_float2(ex2(v.x), ex2(v.y));
                                sum2 = __fadd2_rn(sum2, p);
                                hi[j >> 1] = split2<typename C::H>(p, lo[j >> 1]);
                            }
                        };
                        if (split) {
                            uint32_t w[16], zero[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) zero[j] = 0u;
#pragma unroll
                            for (int kk = 1; kk < 4; ++kk) tmem_st16(sc + 16 * ((quarter + kk) & 3), zero);
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                const float ev = C::kF32 ? exponent(2 * quarter + g) : 0.0f;
                                sum2 = make_float2(0.0f, 0.0f);
                                weigh8(few_x + 8 * g, C::kF32 ? factor(2 * quarter + g) : cq, ev - mref, w + 4 * g,
                                       w + 8 + 4 * g);
                                l = fmaf(sum2.x + sum2.y, C::kF32 ? pow2(-(int)ev) : 1.0f, l);
                            }
                            tmem_st16(sc + 16 * quarter, w);
                        } else if constexpr (C::kF32) {
                            auto weigh = [&](float *y, int kk) {
                                uint32_t w[16];
                                past_end(y, 16 * kk, 16);
#pragma unroll
                                for (int g = 0; g < 2; ++g) {
                                    const float ev = exponent(2 * kk + g);
                                    sum2 = make_float2(0.0f, 0.0f);
                                    weigh8(y + 8 * g, factor(2 * kk + g), ev - mref, w + 4 * g, w + 8 + 4 * g);
                                    l = fmaf(sum2.x + sum2.y, pow2(-(int)ev), l);
                                }
                                tmem_st16(sc + 16 * kk, w);
                            };
                            float xa[16], xb[16];
                            tmem_ld16_nowait(sc, xa);
#pragma unroll 1
                            for (int kk = 0; kk < 4; kk += 2) {
                                tmem_wait_ld();
                                tmem_ld16_nowait(sc + 16 * kk + 16, xb);
                                weigh(xa, kk);
                                tmem_wait_ld();
                                if (kk == 0) tmem_ld16_nowait(sc + 32, xa);
                                weigh(xb, kk + 1);
                            }
                        } else {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                uint32_t w[16];
                                weigh8(x + 16 * kk, cq, -mref, w, w + 8);
                                weigh8(x + 16 * kk + 8, cq, -mref, w + 4, w + 12);
                                tmem_st16(sc + 16 * kk, w);
                            }
                            l += sum2.x + sum2.y;
                        }
                        tmem_wait_st();
                    }
                    wait_pv();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pready[buf]);
                }
                if (stream)
                    ++pv1;
                else
                    ++pv0;
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == C::kSoftWarps) {
        __syncwarp();
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- the rows' partials together, and the rows' weights -----------------------------------------
constexpr int kCombWarps = 8;
constexpr int kCombUnroll = 8;        // partials of a row in flight
constexpr int kMaxGroup = 1024;

// CTA (KV head g, sequence b, z): warps take the group's heads; z = 0 writes
// the outputs, and all z share the rows whose weights are kept.
template <class T, int HD>
__global__ void __launch_bounds__(32 * kCombWarps) attention_combine_kernel(const __grid_constant__ AbArgs a) {
    using C = Cfg<T, HD>;
    constexpr int kVec = C::kDV / 32;     // value columns per lane
    __shared__ float2 stat[kMaxGroup];    // (M, 1 / L) of each head of the group
    const int g = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    const int cum = __ldcg(a.cum + b), places = __ldcg(a.cum + b + 1) - cum;
    const List l(a, C::kNDV, __ldcg(a.cum + a.n_seq));
    const int n_out = blockIdx.z == 0 ? C::kNDV : 1;    // the weights need one half's sums only
    const bool out = blockIdx.z == 0;
    for (int i = warp; i < a.group * n_out; i += kCombWarps) {
        const int hh = i / n_out, dv = i % n_out;
        // the row's partials: a unit's are its CTAs' in turn, `np` prefix ones first
        const int rp = b * a.group + hh;
        const int up = (g * a.m_p + rp / kM) * C::kNDV + dv, uo = (g * a.m_o + hh / kM) * C::kNDV + dv;
        int np = 0, no = 0, cp = 0, co = 0;
        if (l.lt > 0) {
            cp = l.owner(up * l.lt + a.pad);
            np = l.owner(up * l.lt + l.lt - 1) - cp + 1;
        }
        if (places > 0) {
            const int to = l.tp + cum * l.units_o + uo * places;
            co = l.owner(to + a.pad);
            no = l.owner(to + places - 1) - co + 1;
        }
        const size_t r0p = (size_t)(cp + up) * a.rows_p + rp % kM;
        const size_t r0o = (size_t)(co + b * l.units_o + uo) * a.rows_o + hh % kM;
        float M = -INFINITY, L = 0.0f, acc[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) acc[k] = 0.0f;
        float v[kCombUnroll][kVec];
        auto fetch = [&](int k0, int m) {       // O of partials k0 .. k0 + kCombUnroll - 1, m of them there
#pragma unroll
            for (int j = 0; j < kCombUnroll; ++j) {
                const int kk = k0 + j;
                const float *p = kk < np ? a.part_p + (r0p + (size_t)kk * a.rows_p) * C::kDV
                                         : a.part_o + (r0o + (size_t)(kk - np) * a.rows_o) * C::kDV;
#pragma unroll
                for (int q = 0; q < kVec; ++q) v[j][q] = j < m ? __ldcg(p + lane + 32 * q) : 0.0f;
            }
        };
#pragma unroll 1
        for (int k0 = 0; k0 < np + no; k0 += 32) {
            const int k = k0 + lane, m = min(32, np + no - k0);
            float2 x = make_float2(-INFINITY, 0.0f);
            if (k < np)
                x = __ldcg(a.ml_p + r0p + (size_t)k * a.rows_p);
            else if (k < np + no)
                x = __ldcg(a.ml_o + r0o + (size_t)(k - np) * a.rows_o);
            if (out) fetch(k0, m);              // on their way together with (m, l)
            float top = x.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(M, top);
            // (-inf: no score)
            const float f = x.x > -INFINITY ? ex2(x.x - top) : 0.0f, old = M > -INFINITY ? ex2(M - top) : 0.0f;
            M = top;
            L = fmaf(L, old, warp_sum(x.y * f));
            if (!out) continue;
#pragma unroll
            for (int q = 0; q < kVec; ++q) acc[q] *= old;
#pragma unroll 1
            for (int j0 = 0; j0 < m; j0 += kCombUnroll) {
                if (j0) fetch(k0 + j0, m - j0);
#pragma unroll
                for (int j = 0; j < kCombUnroll; ++j) {
                    const float w = __shfl_sync(0xffffffffu, f, (j0 + j) & 31);
#pragma unroll
                    for (int q = 0; q < kVec; ++q) acc[q] = fmaf(v[j][q], w, acc[q]);
                }
            }
        }
        // no rows: 0; rows whose scores are all -inf: 0 / 0, as NaN as a NaN among them
        const float inv = np + no > 0 ? 1.0f / L : 0.0f;
        if (out) {
            T *o = static_cast<T *>(a.out) + ((size_t)b * a.n_head + (size_t)g * a.group + hh) * HD + dv * C::kDV +
                   lane;
#pragma unroll
            for (int k = 0; k < kVec; ++k) o[32 * k] = from_f32<T>(acc[k] * inv);
        }
        if (dv == 0 && lane == 0) stat[hh] = make_float2(M, inv);
    }
    if (!a.add_weights) return;
    __syncthreads();
    const int n = checked_len(a, __ldcg(a.lens + b));
    const float *sc = a.score + ((size_t)b * a.n_head + (size_t)g * a.group) * a.pitch;
    float *w = a.row_weight + ((size_t)b * a.n_kv + g) * a.max_ctx;
    for (int j = blockIdx.z * 32 * kCombWarps + threadIdx.x; j < n; j += gridDim.z * 32 * kCombWarps) {
        float sum = 0.0f;
        for (int hh = 0; hh < a.group; ++hh) {
            const float2 x = stat[hh];
            sum = fmaf(ex2(__ldcg(sc + (size_t)hh * a.pitch + j) - x.x), x.y, sum);
        }
        w[j] = a.decay == 0.0f ? sum : fmaf(a.decay, w[j], sum);
    }
}

// ---- host -----------------------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Shapes, without pointers.
int ab_shape(const lalb_kv_batch *c, const lalb_attn_batch *p) {
    if (int st = kv_batch_shape(c)) return st;
    if (!p || p->prefix_len < 0) return LALB_ERR_INVALID;
    if (int st = lalb_attention_check(p->n_head, c->n_kv_head, c->head_dim)) return st;
    // a row number rounded up to a tile stays in 31 bits
    if (p->prefix_len > (1 << 30) || c->max_ctx > (1 << 30)) return LALB_ERR_UNSUPPORTED;
    const long long group = p->n_head / c->n_kv_head;
    if (group > kMaxGroup || (long long)p->n_head * c->head_dim > (1 << 24) || c->n_seq > 65535 ||
        c->n_kv_head > 65535)
        return LALB_ERR_UNSUPPORTED;
    // places of the list at most, and query rows: 31-bit indices
    const long long mp = (c->n_seq * group + kM - 1) / kM, mo = (group + kM - 1) / kM;
    const long long tiles = 2ll * c->n_kv_head * (mp * places_of(p->prefix_len, kPad16) +
                                                  mo * c->n_seq * (long long)places_of(c->max_ctx, kPad16));
    if (tiles > (1ll << 30) || c->n_seq * group > (1ll << 30)) return LALB_ERR_UNSUPPORTED;
    return LALB_OK;
}

struct Plan {
    AbArgs a;
    size_t o_cum, o_mlp, o_mlo, o_pp, o_po, o_sum, o_score, bytes;
};

void make_plan(const lalb_kv_batch *c, const lalb_attn_batch *p, Plan *pl) {
    AbArgs &a = pl->a;
    a = AbArgs();
    a.n_seq = c->n_seq;
    a.n_head = p->n_head;
    a.n_kv = c->n_kv_head;
    a.group = p->n_head / c->n_kv_head;
    a.max_ctx = c->max_ctx;
    a.prefix = p->prefix_len;
    a.add_weights = p->add_weights != 0;
    const int ndv = c->dtype == LALB_DT_F32 && c->head_dim == 256 ? 2 : 1;   // Cfg::kNDV
    a.m_p = (a.n_seq * a.group + kM - 1) / kM;
    a.m_o = (a.group + kM - 1) / kM;
    a.rows_p = std::min(kM, a.n_seq * a.group);
    a.rows_o = std::min(kM, a.group);
    a.pitch = tiles_of(a.max_ctx) * kTile;
    a.pad = c->dtype == LALB_DT_F32 ? kPadF32 : kPad16;
    const int hd = c->head_dim, dv = hd / ndv;
    // a segment's slot is its CTA's number plus its unit's
    const size_t sp = a.prefix ? (size_t)kGrid + (size_t)a.n_kv * a.m_p * ndv : 0;
    const size_t so = (size_t)kGrid + (size_t)a.n_seq * a.n_kv * a.m_o * ndv;
    size_t off = 0;
    auto take = [&](size_t n) {
        const size_t at = off;
        off += up256(n);
        return at;
    };
    pl->o_cum = take(((size_t)a.n_seq + 1) * sizeof(int));
    pl->o_mlp = take(sp * a.rows_p * sizeof(float2));
    pl->o_mlo = take(so * a.rows_o * sizeof(float2));
    pl->o_pp = take(sp * a.rows_p * dv * sizeof(float));
    pl->o_po = take(so * a.rows_o * dv * sizeof(float));
    // F32: two streams of 128 value columns at most
    pl->o_sum = take(c->dtype == LALB_DT_F32 ? (size_t)kGrid * std::min(2 * hd, 256) * kM * sizeof(float) : 0);
    pl->o_score = take(a.add_weights ? (size_t)a.n_seq * a.n_head * a.pitch * sizeof(float) : 0);
    pl->bytes = off;
}

struct Kernels {
    const void *tiles, *combine;
    int threads, smem, rows;
    int regs;                      // a thread at launch, which the roles' split shares out
    std::atomic<int> *checked;     // the kernel's register count as loaded, once read
};

template <class T, int HD>
Kernels kernels_of() {
    using C = Cfg<T, HD>;
    static std::atomic<int> checked{0};
    return {(const void *)attention_tiles_kernel<T, HD>, (const void *)attention_combine_kernel<T, HD>, C::kThreads,
            (int)C::kSmem, C::kRows, C::kSoftRegs ? C::kEven : 0, &checked};
}

template <class T>
Kernels kernels_for(int hd) {
    switch (hd) {
        case 32: return kernels_of<T, 32>();
        case 64: return kernels_of<T, 64>();
        case 128: return kernels_of<T, 128>();
        default: return kernels_of<T, 256>();
    }
}

}  // namespace

extern "C" int lalb_attention_batch_ws_bytes(const lalb_kv_batch *cache, const lalb_attn_batch *attn,
                                             size_t *bytes) {
    if (!bytes) return LALB_ERR_INVALID;
    if (int st = ab_shape(cache, attn)) return st;
    Plan pl;
    make_plan(cache, attn, &pl);
    *bytes = pl.bytes;
    return LALB_OK;
}

extern "C" int lalb_attention_batch(lalb_ctx *ctx, const lalb_kv_batch *cache, const lalb_attn_batch *attn,
                                    const void *q, long long q_stride, const int32_t *lens, void *ws, void *out,
                                    lalb_stream stream) try {
    if (!ctx) return LALB_ERR_INVALID;
    if (!cache || !attn || !q || !lens || !ws || !out)
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: null pointer");
    if (int st = kv_batch_check(ctx, cache, "attention_batch")) return st;
    if (int st = ab_shape(cache, attn))
        return lalb_fail(ctx, st, "attention_batch: n_head %d over %d KV heads (at most 1024 each), prefix_len %d",
                         attn->n_head, cache->n_kv_head, attn->prefix_len);
    const int es = dtype_size(cache->dtype);
    if (attn->prefix_len > 0 && (!attn->prefix_k || !attn->prefix_v ||
                                 (((uintptr_t)attn->prefix_k | (uintptr_t)attn->prefix_v) & 15u)))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: prefix_k and prefix_v must be 16-byte aligned");
    if (q_stride < (long long)attn->n_head * cache->head_dim || q_stride * es % 16 || ((uintptr_t)q & 15u) ||
        ((uintptr_t)out & 15u) || ((uintptr_t)lens & 3u) || ((uintptr_t)ws & 255u))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: q_stride %lld, or a misaligned buffer", q_stride);
    if (!std::isfinite(attn->scale) || (attn->add_weights && !std::isfinite(attn->decay)))
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: scale and decay must be finite");
    if (attn->add_weights && !cache->row_weight)
        return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: add_weights needs the cache's row_weight");
    Plan pl;
    make_plan(cache, attn, &pl);
    AbArgs &a = pl.a;
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.q = q;
    a.pk = attn->prefix_k;
    a.pv = attn->prefix_v;
    a.k = cache->k;
    a.v = cache->v;
    a.lens = lens;
    a.cum = reinterpret_cast<int *>(w + pl.o_cum);
    a.ml_p = reinterpret_cast<float2 *>(w + pl.o_mlp);
    a.ml_o = reinterpret_cast<float2 *>(w + pl.o_mlo);
    a.part_p = reinterpret_cast<float *>(w + pl.o_pp);
    a.part_o = reinterpret_cast<float *>(w + pl.o_po);
    a.sum = reinterpret_cast<float *>(w + pl.o_sum);
    a.score = reinterpret_cast<float *>(w + pl.o_score);
    a.row_weight = cache->row_weight;
    a.out = out;
    a.status = &ctx->scratch->status;
    a.q_stride = q_stride;
    const double scale = attn->scale == 0.0f ? 1.0 / sqrt((double)cache->head_dim) : (double)attn->scale;
    // kept away from 0, where (masked) -inf x 0 would be NaN
    a.c = (float)std::max(1e-37, fabs(scale) * 1.4426950408889634074);
    if (!std::isfinite(a.c)) return lalb_fail(ctx, LALB_ERR_INVALID, "attention_batch: scale %g", scale);
    a.sign = scale < 0.0 ? -1.0f : 1.0f;
    a.decay = attn->decay;
    DeviceGuard guard(ctx->device);
    if (!guard.ok()) return lalb_fail(ctx, LALB_ERR_CUDA, "attention_batch: device %d", ctx->device);
    const int hd = cache->head_dim;
    const Kernels kn = cache->dtype == LALB_DT_F32   ? kernels_for<float>(hd)
                       : cache->dtype == LALB_DT_F16 ? kernels_for<__half>(hd)
                                                     : kernels_for<__nv_bfloat16>(hd);
    if (int st = lalb_set_smem_attr(ctx, kn.tiles, kn.smem)) return st;
    // a block launched with fewer registers than its roles ask for would wait for them for good
    if (kn.regs) {
        int regs = kn.checked->load(std::memory_order_relaxed);
        if (!regs) {
            cudaFuncAttributes attr;
            LALB_CUDA_TRY(ctx, cudaFuncGetAttributes(&attr, kn.tiles));
            regs = attr.numRegs;
            kn.checked->store(regs, std::memory_order_relaxed);
        }
        if (regs < kn.regs)
            return lalb_fail(ctx, LALB_ERR_UNSUPPORTED, "attention_batch: kernel built with %d registers of %d", regs,
                             kn.regs);
    }
    CUtensorMap maps[4] = {};
    {
        // 16 bits: swizzled 64-column tiles of 64 rows; F32: a loader warp's plain rows of a head
        const CUtensorMapDataType dt = es == 4                         ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : cache->dtype == LALB_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const int box = es == 4 ? hd : std::min(64, hd), rows_box = es == 4 ? kn.rows : kTile;
        const CUtensorMapSwizzle sw = es == 4     ? CU_TENSOR_MAP_SWIZZLE_NONE
                                      : box == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                                  : CU_TENSOR_MAP_SWIZZLE_64B;
        const void *base[4] = {a.pk, a.pv, a.k, a.v};
        for (int i = 0; i < 4; ++i) {
            const long long rows = i < 2 ? a.prefix : (long long)a.n_seq * a.max_ctx;
            if (rows == 0) continue;
            if (int st = map2d(ctx, &maps[i], base[i], dt, es, (long long)a.n_kv * hd, rows, box, rows_box, sw))
                return st;
        }
    }
    if (int st = launch_pdl(ctx, kn.tiles, dim3(kGrid), dim3(kn.threads), kn.smem, (cudaStream_t)stream,
                            {&maps[0], &maps[1], &maps[2], &maps[3], &a}))
        return st;
    LALB_LAUNCH_CHECK(ctx, "attention_tiles_kernel");
    // weights: as many CTAs per (sequence, KV head) as fill the GPU, 1024 rows each at least
    int z = 1;
    if (a.add_weights)
        z = (int)std::max(1ll, std::min<long long>((a.max_ctx + 1023) / 1024,
                                                   (4ll * ctx->sm_count) / ((long long)a.n_seq * a.n_kv)));
    if (int st = launch_pdl(ctx, kn.combine, dim3(a.n_kv, a.n_seq, z), dim3(32 * kCombWarps), 0,
                            (cudaStream_t)stream, {&a}))
        return st;
    LALB_LAUNCH_CHECK(ctx, "attention_combine_kernel");
    return LALB_OK;
} catch (...) {   // out of host memory: no exception leaves a C entry point
    return LALB_ERR_NOMEM;
}
