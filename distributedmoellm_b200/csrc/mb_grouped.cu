// Products of rows grouped by expert with each expert's float matrix (e4m3 with
// block scales, bf16 or f16), and the gate|up form with SiLU(gate) * up.
//
//   y[p, o] = sum_g xs[p, g] ws[e, o / 128, g] sum_{k in g} x[p, k] w[e, o, k]
//
// with g over groups of 128 columns (one group, scales 1, for 16-bit types).
//
// One persistent, warp-specialised kernel on the tcgen05 tensor cores.  The
// rows of x are the M side (128 TMEM lanes, padded), 128 or 256 weight rows the
// N side.  An epilogue thread then owns one row of x: a step's scale is one
// number for all its columns, a row's largest value is found without other
// lanes, and results are runs of a row.  (The other way round, weights as M,
// ragged groups waste no tensor work, but every thread needs every row's scale
// at every step: those shared-memory reads and the stores of single columns
// took 374 us where this takes 279, at 4096 x 14336 x 4096, both since improved.)  A work item is (expert, block of
// weight rows, pass of at most MT rows of x), passes of one block next to each
// other so that its weights come from HBM once; the gate|up form takes 128 gate
// rows and the 128 up rows of the same columns together.
//  * warp 0: TMA loads (128-byte swizzle, K-major) of 128 bytes of every row
//    of the pass and of the weight block, into a ring of stages;
//  * warp 1: tcgen05.mma, f32 accumulators in TMEM.  e4m3 writes each group of
//    128 columns to a fresh accumulator, since the group's two scales differ
//    from the next one's.  16-bit types with 16-bit results accumulate over
//    all of K; with f32 results they start afresh every 256 columns: the tensor
//    cores' f32 sums are cut rather than rounded, which over 2048 columns
//    came to 2.1e-6 of the result (f32 itself: 1e-7);
//  * warp 2 finds the items; warp 3 (e4m3) brings the scales of four steps at a
//    time into shared memory;
//  * warps 4..11: two sets of four (one warp per TMEM lane quarter), each with
//    half of the columns: sums (e4m3: times their scale) into f32 registers
//    while the next columns of K are multiplied, then the results, through
//    shared memory of the warp's own so that they leave as 64-byte runs.  A
//    quarter without rows is skipped.  (Small passes: see Roles.)
// Splitting K: with few items a cluster's CTAs take equal shares of one item's
// groups and send their f32 partial sums through distributed shared memory to
// the first of them, which adds them in rank order, so results do not depend on
// timing.
// Every wait of a role is bounded (status word + abort flag), so each reaches the
// CTA's (and cluster's) barriers at the end, which have no limit of their own.
//
// Measured in bursts of a graph / in a row, where large calls meet the power limit.  Few rows an expert: 512 picks of 128
// e4m3 experts of 2048 x 768, of which they meet about 105, take 34 / 38 us (170 MB of operands and results, 5.0 TB/s; DRAM
// is busy half of the cycles, the rest goes to items of six steps and their hand-overs).  Many: products and epilogue each
// take 160-180 us of the 247 / 288 of 4096 x 14336 x 4096 (e4m3, 1.95 / 1.67 PFLOP/s); 16384 picks of f16 experts of 1536 x
// 2048 take 173 / 210 us (837 MB, 4.8 TB/s), of e4m3 experts of 2048 x 768 80 / 92 (4.3 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mb_common.cuh"
#include "mb_float.cuh"
#include "mb_tc.cuh"

namespace {

// Who does what.  Small passes (at most 32 rows) use one quarter of the TMEM lanes, which the warps 0 and 4 can read: six
// warps, half of the shared and the tensor memory, and so two CTAs per SM, one's hand-overs and prologue beside the
// other's.  Large passes: one CTA per SM, eight epilogue warps; 168 registers a thread at launch, of which the epilogue
// warpgroups (up to 128 sums a thread) take their share from the first: 128 * 72 + 256 * 216 = 64512 = 384 * 168.
// (Sixteen epilogue warps with half the columns each measured the same: a step's length is the round trip from the
// products to the sums and back over the two accumulators that TMEM holds, about 900 cycles.)
template <bool SMALL, bool FP8>
struct Roles {
    static constexpr int kEpiWarps = SMALL ? 2 : 8;
    static constexpr int kWarps = SMALL ? 6 : 12, kThreads = 32 * kWarps;
    static constexpr int kLoad = SMALL ? 1 : 0, kMma = SMALL ? 2 : 1, kFind = SMALL ? 3 : 2, kScale = SMALL ? 5 : 3;
    static constexpr int kTmemCols = SMALL ? 256 : 512;
    static constexpr int kCtas = SMALL ? 2 : 1;            // per SM
    // Tiles of results a warp has in flight.  e4m3 sums wait for the epilogue at every step, so large e4m3 passes send
    // their results by TMA, two tiles while the next two are filled, at the price of the fourth stage (which measured
    // nothing there, and 8% for 16-bit types): 78 us for 16384 picks with f32 results, 89 by vector stores.
    static constexpr int kTiles = !SMALL && FP8 ? 4 : 1;
    static constexpr int kMaxRed = SMALL ? 48 << 10 : 32 << 10;   // shared memory for partial sums of a split
    static constexpr int kMaxSmem = SMALL ? 115712 : 232448;   // 227 KB of 228, or half of 228 less 1 KB
};
constexpr int kLoadRegs = 72, kEpiRegs = 216;
constexpr int kSets = 2;                  // of epilogue warps, each with half of an item's columns
constexpr int kBlock = 128;               // weight rows of a block
constexpr int kTileW = kBlock * 128;      // bytes of a block's tile: 128 rows of 128 bytes
constexpr int kMaxM = 128;                // rows of x per pass
constexpr int kQuarters = 4;              // of the TMEM lanes, 32 rows each
constexpr int kUnit = 4;                  // K steps whose scales are handed over together
constexpr int kScSlots = 3;               // ring of such units
constexpr int kScFloats = kUnit * (128 + 2);   // of each step: xs of the pass's rows, ws of the item's (up to) two blocks
constexpr int kItemSlots = 4;
constexpr int kMaxAcc = 4;
constexpr int kMaxStages = 16;
constexpr int kRowMaps = 4;               // boxes of 16, 32, 64, 128 rows of x
constexpr int kSmallRows = 32;            // rows of a small pass, at most
constexpr int kRun = 64;                  // results leave in runs of 64 bytes a row ..
constexpr int kTile = 32 * kRun;          // .. and tiles of 32 rows
constexpr int kDrainTries = 100000;       // polls for work in flight at a role's end, at most

__device__ unsigned g_no_status;          // where kernels report when the caller gives no status word

struct GroupedArgs {
    const void* x;
    int64_t ldx;
    const float* xs;
    int64_t xs_row, xs_group;
    int64_t P;
    const void* w;
    int64_t w_expert, ldw;
    const float* ws;
    int E, O, K;               // O: output columns (gate|up: I, whose matrices have 2I rows)
    const int32_t* offsets;    // null: one expert, all rows
    void* y;
    int64_t ldy;
    float* qs;
    int64_t qs_row, qs_group;
    unsigned* status;
    int64_t likely;            // rows within the offsets, as far as the host knows: what sizes and splits go by
    int Kb;                    // K steps (128 bytes of a row each)
    int Nb;                    // column blocks of an item's width
    int MT;                    // rows of x per pass, at most
    int stages;
    int prom;                  // K steps summed in TMEM before their sum is added to the f32 registers
    int vec;                   // rows of results start on 16-byte boundaries
};

struct Maps {
    CUtensorMap w;
    CUtensorMap x[kRowMaps];
    CUtensorMap y[2];          // tiles of results: runs of 32 rows, of 8 rows
};

// A work item: expert, block of weight rows, first row of x and how many (none: no more items).
struct Item {
    int e, nb, row0, nrows;
};

// The items of this CTA (of its group of `split` CTAs, when items are split over K) in order.  Finding one takes a search
// and divisions, so one warp does it and hands the items on.
struct Finder {
    const GroupedArgs& a;
    const int2* meta;          // (first row, rows) of each expert
    const int* pstart;         // first item of each expert; [E]: all items
    int it, step, e;
    __device__ Item next()
    {
        it += step;
        if (it >= pstart[a.E]) return {0, 0, 0, 0};
        if (it >= pstart[e + 1]) {         // the last e with pstart[e] <= it (experts without rows have none)
            int lo = e + 1, hi = a.E;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pstart[mid] <= it)
                    lo = mid;
                else
                    hi = mid;
            }
            e = lo;
        }
        const int2 m = meta[e];
        const int passes = (m.y + a.MT - 1) / a.MT;
        const int local = it - pstart[e];
        const int nb = local / passes, pass = local - nb * passes;
        const int size = ((m.y + passes - 1) / passes + 15) & ~15;     // passes of about equal size
        return {e, nb, m.x + pass * size, min(size, m.y - pass * size)};
    }
};

// Where the other roles take the items from.
struct ItemRing {
    const Item* slots;
    uint64_t *full, *empty;
    unsigned* status;
    volatile int* abort_flag;
    Ring r;
    // The next item (of a whole warp, or of one thread alone); false when there is none.
    template <bool WARP>
    __device__ __forceinline__ bool pop(Item& v)
    {
        bool got = mb_mbar_wait_spin(&full[r.slot], r.full_parity(), status, abort_flag);
        if (WARP) got = __all_sync(0xffffffffu, got);      // lanes give up together
        if (!got) return false;
        v = slots[r.slot];
        if (WARP) __syncwarp();
        if (!WARP || (threadIdx.x & 31) == 0) mb_mbar_arrive(&empty[r.slot]);
        r.next();
        return v.nrows > 0;
    }
};

__host__ __device__ constexpr int out_bytes(int out) { return out == MB_T_F32 ? 4 : out == MB_T_E4M3 ? 1 : 2; }

// Two results as 16-bit numbers, packed.
template <int OUT>
__device__ __forceinline__ uint32_t round2(float lo, float hi)
{
    if (OUT == MB_T_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// g / (1 + exp(-g)), by the fast exponential and division (a few units of f32 each, |g| 2^-22 of the exponential's argument
// on top: far below the rounding of any result type).  The fast division gives 0 for divisors from 2^126 on, that is below
// -87.3, where the quotient is still a normal number; from -64 down 1 + exp(-g) is exp(-g) to the last bit, and g exp(g) the
// same quotient.
__device__ __forceinline__ float silu(float g)
{
    const bool low = g < -64.0f;
    const float t = __expf(low ? g : -g);
    return low ? g * t : __fdividef(g, 1.0f + t);
}

// WIDE: an item is two blocks of 128 weight rows, one per epilogue set (gate|up: the gate and the up rows of 128 columns,
// of which each set takes 64); else one block, 64 columns per set.  OUT: the result type (gate|up: TYPE).
template <int TYPE, bool DUAL, bool WIDE, bool SMALL, int OUT>
struct Epilogue {
    static constexpr bool FP8 = TYPE == MB_T_E4M3;
    static constexpr int H = DUAL ? 2 : 1;
    static constexpr int N = WIDE ? 256 : 128;             // accumulator columns of an item
    using Role = Roles<SMALL, FP8>;
    static constexpr int kTiles = Role::kTiles;
    static constexpr int kBatch = kTiles > 1 && OUT != MB_T_E4M3 ? 2 : 1;   // tiles sent together
    static constexpr int S = N / kSets;                    // of them this thread's
    static constexpr int C = S / 16;                       // chunks of 16
    static constexpr int R = S / H;                        // results of this thread
    static constexpr int B = out_bytes(OUT);
    static constexpr int RC = kRun / B;                    // columns of a run

    const GroupedArgs& a;
    unsigned* status;
    volatile int* abort_flag;
    uint32_t tl;               // TMEM address of the warp's lane quarter
    uint32_t acc_full, acc_empty, sc_full, sc_empty;       // shared-memory addresses
    const float* sc;
    float4* red;               // partial sums: [sender][set][S / 4][MT rows]
    uint64_t *red_full, *red_empty;
    float* amax;               // [2][sets][128 rows]
    uint32_t max_full;         // of each quarter: both sets' maxima are there (shared-memory address)
    uint8_t* tiles;            // the warp's tiles of results
    const CUtensorMap* ymaps;
    int split, srank;
    uint32_t leader;
    int q, set, lane;
    Ring ac, scr;
    int sent, abuf, half;

    // Accumulator column of this thread's chunk c.  Gate|up: its first half of chunks are gate columns, then the up
    // columns of the same place.
    __device__ __forceinline__ int column(int c) const
    {
        if (DUAL) return (c >= C / 2 ? kBlock : 0) + R * set + 16 * (c % (C / 2));
        return S * set + 16 * c;
    }

    // One item's K steps k0 .. k1 - 1 and its results.
    __device__ __forceinline__ void item(const Item& w, int k0, int k1)
    {
        const bool rows = 32 * q < w.nrows;                // this quarter has some
        bool ok = true;
        float sum[C][16];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[c][i] = 0.0f;
        if constexpr (FP8) {
            for (int kb = k0; kb < k1; kb += kUnit) {
                // the scales of up to kUnit steps at once, so that a step has little but its sums
                ok = bar_wait(sc_full + 8 * scr.slot, scr.full_parity(), status, abort_flag) && ok;
                const float* from = sc + scr.slot * kScFloats;
                float s[kUnit][H];
#pragma unroll
                for (int u = 0; u < kUnit; ++u) {
                    const float x = from[130 * u + 32 * q + lane];
                    const float2 b = *reinterpret_cast<const float2*>(from + 130 * u + 128);
                    s[u][0] = x * (!DUAL && WIDE && set >= kSets / 2 ? b.y : b.x);
                    if (DUAL) s[u][H - 1] = x * b.y;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(sc_empty + 8 * scr.slot);
                scr.next();
#pragma unroll
                for (int u = 0; u < kUnit; ++u) {
                    if (kb + u >= k1) break;
                    step(sum, s[u], rows, ok);
                }
            }
        } else {
            const float one[H] = {};
            for (int kb = k0; kb < k1; kb += a.prom) step(sum, one, rows, ok);
        }

        if (split > 1) {
            const int me = 32 * q + lane;
            if (srank > 0) {
                // the receiver has read the previous item's sums (the first wait passes at once)
                ok = mbar_wait_cluster(red_empty, (sent & 1) ^ 1, status, abort_flag) && ok;
                ++sent;
                if (rows && ok) {
                    const uint32_t to =
                        cluster_map(mb_smem_addr(red + ((srank - 1) * 2 + set) * (S / 4) * a.MT + me), leader);
                    if (me < a.MT) {
#pragma unroll
                        for (int j = 0; j < S / 4; ++j) {
                            const float* v = &sum[j / 4][4 * (j % 4)];
                            cluster_st4(to + j * a.MT * 16, v[0], v[1], v[2], v[3]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) cluster_arrive(cluster_map(mb_smem_addr(red_full), leader));
                return;
            }
            ok = mbar_wait_cluster(red_full, sent & 1, status, abort_flag) && ok;
            ++sent;
            if (rows && me < a.MT) {
                for (int r = 0; r < split - 1; ++r) {
                    const float4* from = red + (r * 2 + set) * (S / 4) * a.MT + me;
#pragma unroll
                    for (int j = 0; j < S / 4; ++j) {
                        const float4 v = from[j * a.MT];
                        float* to = &sum[j / 4][4 * (j % 4)];
                        to[0] += v.x, to[1] += v.y, to[2] += v.z, to[3] += v.w;
                    }
                }
            }
            __syncwarp();
            if (lane == 0)
                for (int r = 1; r < split; ++r) cluster_arrive(cluster_map(mb_smem_addr(red_empty), leader + r));
        }

        if (!rows) return;
        if constexpr (DUAL) {
#pragma unroll
            for (int c = 0; c < C / 2; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sum[c][i] = silu(sum[c][i]) * sum[c + C / 2][i];
                }
        }
        const int n = __all_sync(0xffffffffu, ok) ? min(32, w.nrows - 32 * q) : 0;  // rows of this quarter to write
        const int64_t row = (int64_t)w.row0 + 32 * q;
        const int col = (DUAL ? w.nb * kBlock : w.nb * N) + R * set;
        if constexpr (OUT == MB_T_E4M3) {
            encode(sum, row, n, w.nb, col);
        } else {
#pragma unroll
            for (int r0 = 0; r0 < R / RC; r0 += kBatch) {
                begin();
#pragma unroll
                for (int r = 0; r < kBatch; ++r)
#pragma unroll
                    for (int j = 0; j < kRun / 16; ++j) {
                        const int i = (r0 + r) * RC + j * (16 / B);
                        const float* v = &sum[i / 16][i % 16];
                        if constexpr (OUT == MB_T_F32)
                            *run(r, lane, j) = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]),
                                                          __float_as_uint(v[2]), __float_as_uint(v[3]));
                        else
                            *run(r, lane, j) = make_uint4(round2<OUT>(v[0], v[1]), round2<OUT>(v[2], v[3]),
                                                          round2<OUT>(v[4], v[5]), round2<OUT>(v[6], v[7]));
                    }
                send(row, n, col + r0 * RC);
            }
        }
    }

    // One accumulator: its sums, times s for e4m3, to the thread's.
    __device__ __forceinline__ void step(float (&sum)[C][16], const float (&s)[H], bool rows, bool& ok)
    {
        ok = bar_wait(acc_full + 8 * ac.slot, ac.full_parity(), status, abort_flag) && ok;
        tc_after();
        if (rows) {
            const uint32_t from = tl + ac.slot * N;
            float d[2][16];                                // the next chunk is on its way while this one is added
            tc_ld16(from + column(0), d[0]);
            tc_wait_ld(d[0]);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float(&v)[16] = d[c & 1], (&next)[16] = d[(c + 1) & 1];
                if (c + 1 < C) tc_ld16(from + column(c + 1), next);
                const float f = s[DUAL && c >= C / 2 ? H - 1 : 0];
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[c][i] = FP8 ? fmaf(v[i], f, sum[c][i]) : sum[c][i] + v[i];
                if (c + 1 < C) tc_wait_ld(next);
            }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty + 8 * ac.slot);
        ac.next();
    }

    // 16 bytes j of row r in tile t of the batch: a row's change places every two rows (the 64-byte swizzle of the y maps),
    // which keeps both the rows' and the runs' accesses on different banks.
    __device__ __forceinline__ uint4* run(int t, int r, int j) const
    {
        return reinterpret_cast<uint4*>(tiles + (2 * half + t) * kTile + r * kRun + ((j ^ (r >> 1 & 3)) << 4));
    }

    // The tiles to be filled next have been read by whoever sent them.
    __device__ __forceinline__ void begin()
    {
        if (kTiles > 1) {
            half ^= 1;
            bulk_wait_read<1>();
        }
        __syncwarp();
    }

    // The batch's tiles, a run next to a run, to rows row .. row + n - 1 of y, from column col on (not past column O).
    __device__ __forceinline__ void send(int64_t row, int n, int col)
    {
        uint8_t* dst = reinterpret_cast<uint8_t*>(a.y) + (row * a.ldy + col) * B;
        int first = 0;                                     // rows before this one go by TMA, which knows where y ends
        if (kTiles > 1) {
            if (a.vec) {
                // a copy per lane: of a tile's 32 rows, or of 8 rows of as many as there are
                first = max(n, 0) & ~7;
                bulk_fence();
                __syncwarp();
                const int t = first == 32 ? lane : lane >> 2, r = first == 32 ? 0 : 8 * (lane & 3);
                if (t < kBatch && r < first && col + t * RC < a.O)
                    tma_store2(first == 32 ? ymaps : ymaps + 1, tiles + (2 * half + t) * kTile + r * kRun, col + t * RC,
                               (int)row + r);
            }
            bulk_commit();
        }
        __syncwarp();
        if (first >= n) return;
        if (a.vec && col + kBatch * RC <= a.O) {
#pragma unroll
            for (int t = 0; t < kBatch; ++t)
#pragma unroll
                for (int i = 0; i < (kTiles > 1 ? 1 : 4); ++i) {
                    const int r = first + 8 * i + (lane >> 2), j = lane & 3;
                    if (r < n) *reinterpret_cast<uint4*>(dst + r * a.ldy * B + t * kRun + 16 * j) = *run(t, r, j);
                }
        } else {
            // one result at a time, neighbours of a row next to each other
            constexpr int W = kBatch * RC;
            using U16 = typename std::conditional<B == 2, uint16_t, uint8_t>::type;
            using U = typename std::conditional<B == 4, uint32_t, U16>::type;
            const int cols = min(W, a.O - col);
#pragma unroll 8
            for (int k = lane; k < 32 * W; k += 32) {
                const int r = k / W, i = k % W;
                if (r >= first && r < n && i < cols)
                    reinterpret_cast<U*>(dst + r * a.ldy * B)[i] =
                        reinterpret_cast<const U*>(run(i / RC, r, i % RC * B / 16))[i % (16 / B)];
            }
        }
    }

    // This thread's R activations of a row as e4m3, the row's scale over them and the other sets'.
    __device__ __forceinline__ void encode(const float (&v)[C][16], int64_t row, int n, int nb, int col)
    {
        float m = 0.0f;
        if (col + R <= a.O) {
#pragma unroll
            for (int i = 0; i < R; ++i) m = fmaxf(m, fabsf(v[i / 16][i % 16]));
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) m = col + i < a.O ? fmaxf(m, fabsf(v[i / 16][i % 16])) : m;
        }
        // The sets meet at an mbarrier, whose waits are bounded: after a wait that ran out one set may have left already.  A
        // set is at most one item ahead of the other, so two buffers do.
        float* am = amax + abuf * kSets * kMaxM + 32 * q + lane;
        am[set * kMaxM] = m;
        __syncwarp();
        if (lane == 0) bar_arrive(max_full + 8 * q);
        if (!__all_sync(0xffffffffu, bar_wait(max_full + 8 * q, abuf, status, abort_flag))) n = 0;
        abuf ^= 1;
#pragma unroll
        for (int s = 0; s < kSets; ++s) m = fmaxf(m, am[s * kMaxM]);
        const Quotient qu(e4m3_scale(m));
        const bool fast = __all_sync(0xffffffffu, qu.fast || lane >= n);
        if (set == 0 && lane < n) a.qs[(row + lane) * a.qs_row + nb * a.qs_group] = qu.s;
        begin();
#pragma unroll
        for (int j = 0; j < R / 16; ++j) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[4] = {v[j][4 * i], v[j][4 * i + 1], v[j][4 * i + 2], v[j][4 * i + 3]};
                if (fast) {
                    quotient4(x, qu.s, qu.r);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = __fdiv_rn(x[k], qu.s);
                }
                u[i] = to_e4m3x2(x[0], x[1]) | to_e4m3x2(x[2], x[3]) << 16;
            }
            *run(0, lane, j) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        send(row, n, col);
    }
};

template <int R>
__device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// The items of experts whose offsets were not all in order: a range that starts before the end of an earlier one is left out,
// so that no row has two writers and the items stay within the count that the launch allowed for.  (A call, which keeps its
// code out of the way of launches whose offsets are in order: 0.06 us of the 6.9 of 120 picks of 16 e4m3 experts.)
__device__ __noinline__ int disjoint_items(int2* meta, int* pstart, int E, int Nb, int MT)
{
    int total = 0;
    for (int e = 0, end = 0; e < E; ++e) {
        const int2 m = meta[e];
        const int n = m.x < end ? 0 : m.y;
        if (n < m.y) meta[e].y = 0;
        if (n > 0) end = m.x + n;
        pstart[e] = total;
        total += Nb * ((n + MT - 1) / MT);
    }
    return total;
}

template <int TYPE, bool DUAL, bool WIDE, bool SMALL, int OUT>
__global__ void __launch_bounds__(Roles<SMALL, TYPE == MB_T_E4M3>::kThreads, Roles<SMALL, TYPE == MB_T_E4M3>::kCtas)
    grouped_kernel(const __grid_constant__ GroupedArgs a, const __grid_constant__ Maps maps)
{
    using Epi = Epilogue<TYPE, DUAL, WIDE, SMALL, OUT>;
    using Role = typename Epi::Role;
    constexpr int kThreads = Role::kThreads, kWarps = Role::kWarps, kEpiWarps = Role::kEpiWarps;
    constexpr bool FP8 = TYPE == MB_T_E4M3;
    constexpr int KS = FP8 ? 128 : 64;    // columns of a K step
    constexpr int NB = WIDE ? 2 : 1;      // weight tiles of a step
    constexpr int kAcc = Role::kTmemCols / Epi::N;

    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    // a stage: the pass's rows, then the weight tiles.  The products always read 128 rows: past MT they find the weight
    // tiles' bytes, whose results stay in lanes that nobody reads.
    const int stage_bytes = a.MT * 128 + NB * kTileW;
    const uint32_t csize = cluster_size();
    uint8_t* stage0 = smem;
    float4* red = reinterpret_cast<float4*>(stage0 + (size_t)a.stages * stage_bytes);
    uint8_t* tiles = reinterpret_cast<uint8_t*>(red + (csize - 1) * Epi::N / 4 * a.MT);   // 1024-byte aligned
    float* amax = reinterpret_cast<float*>(tiles + kEpiWarps * Epi::kTiles * kTile);
    float* sc = amax + (OUT == MB_T_E4M3 ? 2 * kSets * kMaxM : 0);
    uint64_t* full = reinterpret_cast<uint64_t*>(sc + (FP8 ? kScSlots * kScFloats : 0));
    uint64_t* empty = full + kMaxStages;
    uint64_t* acc_full = empty + kMaxStages;
    uint64_t* acc_empty = acc_full + kMaxAcc;
    uint64_t* sc_full = acc_empty + kMaxAcc;
    uint64_t* sc_empty = sc_full + kScSlots;
    uint64_t* item_full = sc_empty + kScSlots;
    uint64_t* item_empty = item_full + kItemSlots;
    uint64_t* red_full = item_empty + kItemSlots;
    uint64_t* red_empty = red_full + 1;
    uint64_t* max_full = red_empty + 1;
    uint64_t* mma_done = max_full + kQuarters;
    Item* items = reinterpret_cast<Item*>(mma_done + 2);               // 16-byte aligned
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + kItemSlots);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* wsum = reinterpret_cast<int*>(tmem_slot + 2);                 // [kWarps], [31]: split
    int2* meta = reinterpret_cast<int2*>(wsum + 32);                   // [E]
    int* pstart = reinterpret_cast<int*>(meta + a.E);                  // [E + 1]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned* const status = a.status ? a.status : &g_no_status;

    mb_pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            mb_mbar_init(&full[i], 1);
            mb_mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < kAcc; ++i) {
            mb_mbar_init(&acc_full[i], 1);
            mb_mbar_init(&acc_empty[i], kEpiWarps);
        }
        for (int i = 0; i < kScSlots; ++i) {
            mb_mbar_init(&sc_full[i], 1);
            mb_mbar_init(&sc_empty[i], kEpiWarps);
        }
        for (int i = 0; i < kItemSlots; ++i) {
            mb_mbar_init(&item_full[i], 1);
            mb_mbar_init(&item_empty[i], kEpiWarps + (FP8 ? 3 : 2));
        }
        for (int i = 0; i < kQuarters; ++i) mb_mbar_init(&max_full[i], kSets);
        mb_mbar_init(mma_done, 1);
        *abort_flag = 0;
    }
    if (warp == Role::kLoad && lane < 1 + kRowMaps && (lane == 0 || 8 << lane <= a.MT))
        tma_prefetch_map(lane == 0 ? &maps.w : &maps.x[lane - 1]);
    if (warp == Role::kMma) tc_alloc(tmem_slot, Role::kTmemCols);
    mb_pdl_wait();

    // The experts' rows and the first item of each: an exclusive scan over the experts, a run of them per thread.
    {
        const int per = (a.E + kThreads - 1) / kThreads;
        const int e0 = min(a.E, (int)threadIdx.x * per), e1 = min(a.E, e0 + per);
        int mine = 0, bad = 0;
        for (int e = e0; e < e1; ++e) {
            int lo = 0, n = (int)a.P;
            if (a.offsets) {
                lo = a.offsets[e];
                const int hi = a.offsets[e + 1];
                n = hi - lo;
                if (lo < 0 || hi < lo || hi > a.P) {
                    atomicOr(status, MB_STATUS_BADARG);
                    bad = 1;
                    lo = n = 0;
                }
            }
            meta[e] = make_int2(lo, n);
            pstart[e] = mine;
            mine += a.Nb * ((n + a.MT - 1) / a.MT);
        }
        int run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += t;
        }
        if (lane == 31) wsum[warp] = run;
        // Where no pair of offsets decreases, the ranges are disjoint.  Else what is left of them may overlap.
        bad = __syncthreads_or(bad);
        int before = run - mine, total = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int s = wsum[w];
            if (w < warp) before += s;
            total += s;
        }
        if (bad) {
            if (threadIdx.x == 0) total = disjoint_items(meta, pstart, a.E, a.Nb, a.MT);
        } else {
            for (int e = e0; e < e1; ++e) pstart[e] += before;
        }
        if (threadIdx.x == 0) {
            pstart[a.E] = total;
            // How many CTAs share an item: the split whose longest CTA has the fewest K steps, two more for each
            // item that is split (the partial sums' way to the first CTA).
            int64_t best = (int64_t)1 << 62;
            int split = 1;
            for (int s = 1; s <= (int)csize && s <= a.Kb; s <<= 1) {
                const int groups = gridDim.x / s;
                const int64_t c = (int64_t)((total + groups - 1) / groups) * ((a.Kb + s - 1) / s + (s > 1 ? 2 : 0));
                if (c < best) {
                    best = c;
                    split = s;
                }
            }
            wsum[31] = split;
            mb_mbar_init(red_full, kEpiWarps * max(split - 1, 1));
            mb_mbar_init(red_empty, kEpiWarps);
            mb_fence_mbar_init();
        }
    }
    tc_before();
    __syncthreads();
    if (csize > 1) cluster_sync();        // the other CTAs' barriers exist
    tc_after();

    const uint32_t tmem = *tmem_slot;
    const int split = wsum[31];
    const int srank = (int)blockIdx.x % split;                          // rank among the CTAs of an item
    const int k0 = (int)((int64_t)a.Kb * srank / split), k1 = (int)((int64_t)a.Kb * (srank + 1) / split);
    ItemRing ring{items, item_full, item_empty, status, abort_flag, Ring(kItemSlots)};
    Item w;

    if (!SMALL && warp < 4) setmaxnreg_dec<kLoadRegs>();
    if (warp == Role::kLoad) {
        // ------------------------------------------------------------------ loads
        if (elect_one()) {
            Ring st(a.stages);
            bool ok = true;
            int issued = 0;
            const uint32_t stage0s = mb_smem_addr(stage0), fullb = mb_smem_addr(full), emptyb = mb_smem_addr(empty);
            while (ok && ring.pop<false>(w)) {
                const int r16 = (w.nrows + 15) >> 4;
                const uint32_t bytes = NB * kTileW + r16 * 16 * 128;
                for (int kb = k0; kb < k1; ++kb, st.next()) {
                    ok = bar_wait(emptyb + 8 * st.slot, st.empty_parity(), status, abort_flag);
                    if (!ok) break;
                    const uint32_t dst = stage0s + st.slot * stage_bytes, bar = fullb + 8 * st.slot;
                    bar_expect(bar, bytes);
                    tma_load3(dst + a.MT * 128, &maps.w, kb * KS, DUAL ? w.nb * kBlock : w.nb * Epi::N, w.e, bar);
                    if (DUAL)
                        tma_load3(dst + a.MT * 128 + kTileW, &maps.w, kb * KS, a.O + w.nb * kBlock, w.e, bar);
                    int row = 0;                           // boxes of 128, 64, 32, 16 rows: those that add up to the pass's
#pragma unroll
                    for (int b = kRowMaps - 1; b >= 0; --b)
                        if (r16 >> b & 1) {
                            tma_load2(dst + row * 128, &maps.x[b], kb * KS, w.row0 + row, bar);
                            row += 16 << b;
                        }
                    ++issued;
                }
            }
            // The last copies land (bounded) before the CTA may end, whoever gave up and whenever: without that they are what
            // the products have waited for anyway.
            for (int i = 0; i < min(issued, a.stages); ++i) {
                if (--st.slot < 0) {
                    st.slot = a.stages - 1;
                    st.phase ^= 1;
                }
                for (int n = 0; n < kDrainTries && !bar_try(fullb + 8 * st.slot, st.full_parity()); ++n) {
                }
            }
        }
        __syncwarp();
    } else if (warp == Role::kMma) {
        // ------------------------------------------------------------------ tensor cores
        if (elect_one()) {
            Ring st(a.stages), ac(kAcc);
            bool ok = true;
            // M = 128, N, D f32; A and B both K-major: e4m3 / f16 are format 0, bf16 is 1
            constexpr uint32_t idesc = (1u << 4) | (TYPE == MB_T_BF16 ? (1u << 7) | (1u << 10) : 0u) |
                                       ((uint32_t)(Epi::N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint64_t desc0 = tc_desc_sw128(mb_smem_addr(stage0));
            const uint32_t fullb = mb_smem_addr(full), accb = mb_smem_addr(acc_empty);
            const uint32_t step_w = a.MT * 128 >> 4, step_stage = stage_bytes >> 4;
            while (ok && ring.pop<false>(w)) {
                int part = 0;                              // K steps already in the accumulator
                for (int kb = k0; kb < k1; ++kb, st.next()) {
                    if (part == 0) ok = bar_wait(accb + 8 * ac.slot, ac.empty_parity(), status, abort_flag);
                    ok = ok && bar_wait(fullb + 8 * st.slot, st.full_parity(), status, abort_flag);
                    if (!ok) break;
                    tc_after();
                    const uint64_t dx = desc0 + st.slot * step_stage, dw = dx + step_w;
                    const uint32_t d = tmem + ac.slot * Epi::N;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        tc_mma_ss<FP8>(d, dx + 2 * j, dw + 2 * j, idesc, (j > 0 || part > 0) ? 1u : 0u);
                    tc_commit(&empty[st.slot]);
                    if (FP8 || ++part == a.prom || kb + 1 == k1) {
                        tc_commit(&acc_full[ac.slot]);
                        ac.next();
                        part = 0;
                    }
                }
            }
            // so do the products, before TMEM and the barriers that they arrive on go
            tc_commit(mma_done);
            for (int n = 0; n < kDrainTries && !bar_try(mb_smem_addr(mma_done), 0); ++n) {
            }
        }
        __syncwarp();
    } else if (warp == Role::kFind) {
        // ------------------------------------------------------------------ items
        Finder find{a, meta, pstart, (int)blockIdx.x / split - (int)gridDim.x / split, (int)gridDim.x / split, 0};
        Ring r(kItemSlots);
        for (bool more = true; more; r.next()) {
            const Item v = find.next();
            more = v.nrows > 0;
            if (!__all_sync(0xffffffffu, mb_mbar_wait_spin(&item_empty[r.slot], r.empty_parity(), status, abort_flag)))
                break;
            if (lane == 0) {
                items[r.slot] = v;
                mb_mbar_arrive(&item_full[r.slot]);
            }
        }
    } else if (warp == Role::kScale) {
        // ------------------------------------------------------------------ scales
        if (FP8) {
            const int Ob = (a.O + kScaleBlock - 1) / kScaleBlock;
            Ring slot(kScSlots);
            bool ok = true;
            while (ok && ring.pop<true>(w)) {
                // lanes 0, 1: the item's two blocks of weight rows (the last item of an odd count has one)
                const int block = DUAL ? (w.e * 2 + (lane & 1)) * Ob + w.nb
                                       : w.e * Ob + min(NB * w.nb + (WIDE ? lane & 1 : 0), Ob - 1);
                const float* wsp = a.ws + (int64_t)block * a.Kb;
                const float* xsp = a.xs + ((int64_t)w.row0 + lane) * a.xs_row;
                for (int kb = k0; kb < k1; kb += kUnit) {
                    float v[kUnit][4], b[kUnit];
#pragma unroll
                    for (int s = 0; s < kUnit; ++s) {
                        const bool real = kb + s < k1;
                        b[s] = real ? wsp[kb + s] : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            v[s][i] = real && lane + 32 * i < w.nrows
                                          ? xsp[(int64_t)(32 * i) * a.xs_row + (int64_t)(kb + s) * a.xs_group]
                                          : 0.0f;
                    }
                    ok = __all_sync(0xffffffffu, mb_mbar_wait_spin(&sc_empty[slot.slot], slot.empty_parity(), status,
                                                                  abort_flag));
                    if (!ok) break;
                    float* dst = sc + slot.slot * kScFloats;
#pragma unroll
                    for (int s = 0; s < kUnit; ++s) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (32 * i < w.nrows) dst[s * 130 + lane + 32 * i] = v[s][i];
                        if (lane < 2) dst[s * 130 + 128 + lane] = b[s];
                    }
                    __syncwarp();
                    if (lane == 0) mb_mbar_arrive(&sc_full[slot.slot]);
                    slot.next();
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        if (!SMALL) setmaxnreg_inc<kEpiRegs>();
        const int q = warp & 3, set = SMALL ? warp >> 2 : (warp >> 2) - 1;
        Epi ep{a, status, abort_flag, tmem + ((uint32_t)(32 * q) << 16), mb_smem_addr(acc_full),
               mb_smem_addr(acc_empty), mb_smem_addr(sc_full), mb_smem_addr(sc_empty), sc, red,
               red_full, red_empty, amax, mb_smem_addr(max_full), tiles + (SMALL ? set : warp - 4) * Epi::kTiles * kTile, maps.y, split, srank,
               cluster_rank() - srank, q, set, lane, Ring(kAcc), Ring(kScSlots), 0, 0, 0};
        while (ring.pop<true>(w)) ep.item(w, k0, k1);
        if (Epi::kTiles > 1) bulk_wait();
    }

    tc_before();
    __syncthreads();
    tc_after();
    if (warp == Role::kMma) tc_dealloc(tmem, Role::kTmemCols);
    if (csize > 1) cluster_sync();        // no CTA ends while another may still write to it
}

// ---- host side -----------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn()
{
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

CUtensorMapDataType map_type(int type)
{
    return type == MB_T_E4M3  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
           : type == MB_T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
           : type == MB_T_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

int elem_bytes(int type) { return type == MB_T_F32 ? 4 : type == MB_T_E4M3 ? 1 : 2; }

// What every product requires of its arguments (halves: 2 for gate|up).  Sizes first: with no rows the pointers may be
// null.
int check_args(const GroupedArgs& a, int type, int halves, const char* what)
{
    MB_REQUIRE(type == MB_T_E4M3 || type == MB_T_BF16 || type == MB_T_F16, "%s: operand type %d", what, type);
    MB_REQUIRE(a.E >= 1 && a.E <= 1024 && a.O >= 1 && a.O <= (1 << 24) && a.K >= 1 && a.K <= (1 << 24) && a.P >= 0 &&
                   a.P < (1ll << 31),
               "%s: E=%d O=%d K=%d P=%lld", what, a.E, a.O, a.K, (long long)a.P);
    MB_REQUIRE(a.likely >= 0 && a.likely <= a.P, "%s: %lld picks of %lld rows", what, (long long)a.likely, (long long)a.P);
    const int64_t b = elem_bytes(type);
    MB_REQUIRE(a.ldx >= a.K && a.ldw >= a.K && a.ldy >= a.O, "%s: rows closer than their width (%lld, %lld, %lld)",
               what, (long long)a.ldx, (long long)a.ldw, (long long)a.ldy);
    MB_REQUIRE(a.E == 1 || a.w_expert >= (int64_t)(halves * a.O - 1) * a.ldw + a.K, "%s: experts' matrices overlap",
               what);
    MB_REQUIRE(a.ldx * b % 16 == 0 && a.ldw * b % 16 == 0 && (a.E == 1 || a.w_expert * b % 16 == 0),
               "%s: rows and matrices must lie a multiple of 16 bytes apart (ldx=%lld ldw=%lld w_expert=%lld)", what,
               (long long)a.ldx, (long long)a.ldw, (long long)a.w_expert);
    if (a.P == 0) return MB_OK;
    MB_REQUIRE(a.x && a.w && a.y && (a.offsets || a.E == 1), "%s: null pointer", what);
    MB_REQUIRE(((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.w & 15) == 0, "%s: x and w must be 16-byte aligned", what);
    MB_REQUIRE(type != MB_T_E4M3 || (a.xs && a.ws), "%s: e4m3 operands need their scales", what);
    return MB_OK;
}

int make_maps(const GroupedArgs& a, int type, int halves, int wrows, int out, bool tiles, Maps* m, const char* what)
{
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return mb_fail(MB_ECUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
    const cuuint64_t b = (cuuint64_t)elem_bytes(type);
    const cuuint32_t inner = (cuuint32_t)(128 / b), one[3] = {1, 1, 1};
    const cuuint64_t wd[3] = {(cuuint64_t)a.K, (cuuint64_t)a.O * halves, (cuuint64_t)a.E};
    const cuuint64_t wst[2] = {(cuuint64_t)a.ldw * b,
                               (cuuint64_t)(a.E > 1 ? a.w_expert : (int64_t)a.O * halves * a.ldw) * b};
    const cuuint32_t wbox[3] = {inner, (cuuint32_t)wrows, 1};
    CUresult r = fn(&m->w, map_type(type), 3, const_cast<void*>(a.w), wd, wst, wbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    const cuuint64_t xd[2] = {(cuuint64_t)a.K, (cuuint64_t)a.P};
    const cuuint64_t xst[1] = {(cuuint64_t)a.ldx * b};
    for (int i = 0; i < kRowMaps && (16 << i) <= a.MT && r == CUDA_SUCCESS; ++i) {
        const cuuint32_t xbox[2] = {inner, (cuuint32_t)(16 << i)};
        r = fn(&m->x[i], map_type(type), 2, const_cast<void*>(a.x), xd, xst, xbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (tiles && a.vec) {
        const cuuint64_t ob = (cuuint64_t)out_bytes(out);
        const cuuint64_t yd[2] = {(cuuint64_t)a.O, (cuuint64_t)a.P}, yst[1] = {(cuuint64_t)a.ldy * ob};
        for (int i = 0; i < 2 && r == CUDA_SUCCESS; ++i) {
            const cuuint32_t ybox[2] = {(cuuint32_t)(kRun / ob), i == 0 ? 32u : 8u};
            r = fn(&m->y[i], map_type(out), 2, a.y, yd, yst, ybox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        }
    }
    if (r != CUDA_SUCCESS) return mb_fail(MB_ECUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return MB_OK;
}

int pow2_at_least(int64_t n, int lo, int hi)
{
    int p = lo;
    while (p < n && p < hi) p <<= 1;
    return p;
}

template <int TYPE, bool DUAL, bool WIDE, bool SMALL, int OUT>
int launch(GroupedArgs a, const char* what, cudaStream_t st)
{
    constexpr bool FP8 = TYPE == MB_T_E4M3;
    constexpr int N = WIDE ? 256 : 128;
    using Role = Roles<SMALL, FP8>;
    const int slots = mb_num_sms() * Role::kCtas;
    const int64_t active = std::min<int64_t>(a.E, a.P);          // experts with rows, at most
    a.Kb = (a.K + (FP8 ? 127 : 63)) / (FP8 ? 128 : 64);
    a.Nb = DUAL ? (a.O + kBlock - 1) / kBlock : (a.O + N - 1) / N;
    a.prom = FP8 ? 1 : OUT == MB_T_F32 ? 4 : a.Kb;
    a.vec = ((uintptr_t)a.y & 15) == 0 && a.ldy * out_bytes(OUT) % 16 == 0;
    const int64_t items = a.Nb * (active + a.P / a.MT);            // an upper bound
    MB_REQUIRE(items < (1ll << 30), "%s: %lld work items", what, (long long)items);
    int cluster = 1;
    if (!(WIDE && !SMALL)) {
        // The split with the fewest K steps in turn on the busiest CTA, the launch of clusters counted as steps too (it
        // measured 1, 3 and 6 us for 2, 4 and 8 CTAs of small passes, a step 0.35 us; passes of 64 rows have more sums to
        // send, and with 128 rows the split lost: 17.8 us against 16.0 at 128 x 4096 x 4096).  Clusters get one CTA per
        // SM, which is what the occupancy query grants them.  Experts with rows: those that the picks meet, each expert as
        // likely as another.
        const double meet = a.offsets ? a.E * (1.0 - std::pow(1.0 - 1.0 / a.E, (double)a.likely)) : 1.0;
        const double passes = std::max(meet, (double)((a.likely + a.MT - 1) / a.MT));
        const int64_t likely = std::max<int64_t>(1, (int64_t)(a.Nb * passes + 0.5));
        int64_t best = (int64_t)1 << 62;
        for (int c = 1, extra = 0; c <= 8 && c <= a.Kb && (c - 1) * N * a.MT * 4 <= Role::kMaxRed; c *= 2) {
            const int64_t groups = (c == 1 ? slots : slots / Role::kCtas) / c;
            const int64_t cost = (likely + groups - 1) / groups * ((a.Kb + c - 1) / c + (c > 1 ? 2 : 0)) + extra;
            if (cost < best) {
                best = cost;
                cluster = c;
            }
            extra = c == 1 ? (SMALL ? 3 : 9) : 2 * extra + 3;
        }
    }
    const int stage = a.MT * 128 + N * 128;
    const int fixed = 1024 + (OUT == MB_T_E4M3 ? 2 * kSets * kMaxM * 4 : 0) + (FP8 ? kScSlots * kScFloats * 4 : 0) +
                      Role::kEpiWarps * Role::kTiles * kTile +
                      (2 * kMaxStages + 2 * kMaxAcc + 2 * kScSlots + 2 * kItemSlots + 2 + kQuarters + 2) * 8 + kItemSlots * 16 + 8 + 128 +
                      a.E * 8 + (a.E + 1) * 4 + 16;
    // a split's partial sums may leave too few stages beside the tables of very many experts: then a smaller split
    while (cluster > 1 && (Role::kMaxSmem - fixed - (cluster - 1) * N * a.MT * 4) / stage < 2) cluster /= 2;
    const int used = fixed + (cluster - 1) * N * a.MT * 4;
    a.stages = std::min(kMaxStages, (Role::kMaxSmem - used) / stage);
    const int smem = used + a.stages * stage;

    auto kern = grouped_kernel<TYPE, DUAL, WIDE, SMALL, OUT>;
    static thread_local uint64_t ready = 0;                        // devices whose attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(ready >> (dev & 63) & 1)) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Role::kMaxSmem);
        if (e == cudaSuccess)             // two small CTAs per SM, clusters of them included, need all of it
            e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return mb_fail(MB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
        ready |= 1ull << (dev & 63);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = Role::kThreads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    int ctas = slots;
    if (cluster > 1) {
        // clusters that fit at the same time: a cluster stays within one GPC
        static thread_local int fits[64][4] = {};
        int& f = fits[dev & 63][cluster == 2 ? 1 : cluster == 4 ? 2 : 3];
        if (f == 0) {
            cfg.gridDim = cluster;
            int n = 0;
            const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
            if (e != cudaSuccess) return mb_fail(MB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
            f = std::max(1, n);
        }
        ctas = f * cluster;
    }
    cfg.gridDim = (unsigned)std::min<int64_t>(ctas, items * cluster);
    Maps maps;
    const int rc = make_maps(a, TYPE, DUAL ? 2 : 1, DUAL ? kBlock : N, OUT, Role::kTiles > 1, &maps, what);
    if (rc) return rc;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps);
    if (e != cudaSuccess) return mb_fail(MB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
    return MB_OK;
}

// Rows per pass: half as many again as an expert has on average (loads differ), as a power of two.  Up to 32 is a small
// pass (us, small / of 64 rows: 512 picks of 128 e4m3 experts 33.2 / 38.9, gate|up of 64 picks 31.6 / 34.6, 8 bf16 picks
// 15.7 / 14.9).
int pass_rows(const GroupedArgs& a)
{
    return pow2_at_least(a.offsets ? (a.likely * 3 / 2 + a.E - 1) / a.E : a.P, 16, kMaxM);
}

// Blocks of 256 weight rows where that still gives every SM an item, else of 128: the wider items move fewer bytes of x
// per product (us, 256 / 128: 16384 picks of 128 e4m3 experts 78 / 86, f16 178 / 194), the narrower ones spread small
// calls over more SMs.
bool wide(const GroupedArgs& a)
{
    const int64_t active = std::min<int64_t>(a.E, a.likely);
    return (a.O + 255) / 256 * (active + a.likely / a.MT) >= mb_num_sms();
}

template <int TYPE, int OUT>
int launch_width(GroupedArgs a, const char* what, cudaStream_t st)
{
    a.MT = pass_rows(a);
    if (a.MT <= kSmallRows) return launch<TYPE, false, false, true, OUT>(a, what, st);
    return wide(a) ? launch<TYPE, false, true, false, OUT>(a, what, st)
                   : launch<TYPE, false, false, false, OUT>(a, what, st);
}

template <int TYPE>
int launch_swiglu(GroupedArgs a, const char* what, cudaStream_t st)
{
    a.MT = pass_rows(a);
    return a.MT <= kSmallRows ? launch<TYPE, true, true, true, TYPE>(a, what, st)
                              : launch<TYPE, true, true, false, TYPE>(a, what, st);
}

template <int TYPE>
int launch_as(const GroupedArgs& a, int y_type, const char* what, cudaStream_t st)
{
    if (y_type == MB_T_F32) return launch_width<TYPE, MB_T_F32>(a, what, st);
    if (y_type == MB_T_BF16) return launch_width<TYPE, MB_T_BF16>(a, what, st);
    return launch_width<TYPE, MB_T_F16>(a, what, st);
}

int matmul(const GroupedArgs& a, int type, int y_type, const char* what, void* stream)
{
    MB_REQUIRE(y_type == MB_T_F32 || y_type == MB_T_BF16 || y_type == MB_T_F16, "%s: result type %d", what, y_type);
    const int rc = check_args(a, type, 1, what);
    if (rc || a.P == 0) return rc;
    const cudaStream_t st = mb_stream(stream);
    if (type == MB_T_E4M3) return launch_as<MB_T_E4M3>(a, y_type, what, st);
    if (type == MB_T_BF16) return launch_as<MB_T_BF16>(a, y_type, what, st);
    return launch_as<MB_T_F16>(a, y_type, what, st);
}

}  // namespace

extern "C" int mb_grouped_matmul_t_slice(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                         int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                         const float* ws, int E, int O, int K, const int32_t* offsets, void* y,
                                         int y_type, int64_t ldy, int64_t picks, unsigned* status, void* stream)
{
    MB_REQUIRE(offsets || P == 0, "mb_grouped_matmul_t: null pointer");
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, O, K,
                        offsets, y, ldy, nullptr, 0, 0, status, picks};
    return matmul(a, type, y_type, "mb_grouped_matmul_t", stream);
}

extern "C" int mb_grouped_matmul_t(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                   int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                   const float* ws, int E, int O, int K, const int32_t* offsets, void* y, int y_type,
                                   int64_t ldy, unsigned* status, void* stream)
{
    return mb_grouped_matmul_t_slice(x, type, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, O, K, offsets, y,
                                     y_type, ldy, P, status, stream);
}

extern "C" int mb_matmul_t_e4m3(const void* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_group,
                                int64_t n, const void* w, int64_t ldw, const float* ws, int O, int K, void* y,
                                int y_type, int64_t ldy, unsigned* status, void* stream)
{
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, n, w, 0, ldw, ws, 1, O, K,
                        nullptr, y, ldy, nullptr, 0, 0, status, n};
    return matmul(a, MB_T_E4M3, y_type, "mb_matmul_t_e4m3", stream);
}

extern "C" int mb_grouped_swiglu_t_slice(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                         int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                         const float* ws, int E, int I, int K, const int32_t* offsets, void* q,
                                         int64_t ldq, float* qs, int64_t qs_row, int64_t qs_group, int64_t picks,
                                         unsigned* status, void* stream)
{
    const char* what = "mb_grouped_swiglu_t";
    MB_REQUIRE(offsets || P == 0, "%s: null pointer", what);
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, I, K,
                        offsets, q, ldq, qs, qs_row, qs_group, status, picks};
    int rc = check_args(a, type, 2, what);
    if (rc || P == 0) return rc;
    MB_REQUIRE(type != MB_T_E4M3 || qs, "%s: e4m3 results need their scales", what);
    const cudaStream_t st = mb_stream(stream);
    if (type == MB_T_E4M3) return launch_swiglu<MB_T_E4M3>(a, what, st);
    if (type == MB_T_BF16) return launch_swiglu<MB_T_BF16>(a, what, st);
    return launch_swiglu<MB_T_F16>(a, what, st);
}

extern "C" int mb_grouped_swiglu_t(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                   int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                   const float* ws, int E, int I, int K, const int32_t* offsets, void* q, int64_t ldq,
                                   float* qs, int64_t qs_row, int64_t qs_group, unsigned* status, void* stream)
{
    return mb_grouped_swiglu_t_slice(x, type, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, I, K, offsets, q,
                                     ldq, qs, qs_row, qs_group, P, status, stream);
}
