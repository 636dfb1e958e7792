// Products of rows grouped by expert with each expert's float matrix (e4m3 with
// block scales, bf16 or f16), and the gate|up form with SiLU(gate) * up.
//
//   y[p, o] = sum_g xs[p, g] ws[e, o / 128, g] sum_{k in g} x[p, k] w[e, o, k]
//
// with g over groups of 128 columns (one group, scales 1, for 16-bit types).
//
// One persistent, warp-specialised kernel on the tcgen05 tensor cores.  The
// weights are the M = 128 side and the rows of x the N side: an expert's row
// count is ragged, N goes in steps of 16 and costs in proportion, and a decode
// step's few rows leave the shared memory to a deep ring of weight tiles.  A
// work item is (expert, block of 128 weight rows, pass of at most NT rows of
// x), passes of one block next to each other so that its weights come from HBM
// once; the gate|up form takes the 128 gate rows and the 128 up rows of the
// same columns together.
//  * warp 0: TMA loads (128-byte swizzle, K-major) of 128 bytes of every row
//    of the weight block and of the pass's rows, into a ring of stages;
//  * warp 1: tcgen05.mma, f32 accumulators in TMEM.  e4m3 writes each group of
//    128 columns to a fresh accumulator, since the group's two scales differ
//    from the next one's.  16-bit types with 16-bit results accumulate over
//    all of K; with f32 results they start afresh every 256 columns: the tensor
//    cores' f32 sums are cut rather than rounded, which over 2048 columns
//    came to 2.1e-6 of the result (f32 itself: 1e-7);
//  * warps 2, 3 (e4m3): xs * ws of each row and group into shared memory, four
//    groups at a time;
//  * warps 4..11: the accumulators' columns, 32 at a time and alternating
//    between two sets of four warps (one set alone for passes of 32 rows or
//    fewer), added (e4m3: times their scale) to f32 registers (packed f32x2
//    operations) while the next columns of K are multiplied.  They are read as
//    16 x 256-bit fragments: a thread then meets 8 rows of x in 32, and needs
//    8 scales from shared memory where whole TMEM rows need all 32 (at 256 rows
//    those reads alone took 1024 cycles a step, twice the products).  Results go
//    through shared memory and leave as whole rows by bulk copies.
// Splitting K: with few items a cluster's CTAs take equal shares of one item's
// groups and send their f32 partial sums through distributed shared memory to
// the first of them, which adds them in rank order, so results do not depend on
// timing.
// Every wait is bounded (status word + abort flag).
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <mutex>

#include "mb_common.cuh"
#include "mb_float.cuh"
#include "mb_tc.cuh"

namespace {

constexpr int kBM = 128;                  // weight rows of a tile = TMEM lanes
constexpr int kThreads = 384;
constexpr int kThreadWarps = kThreads / 32;
constexpr int kEpiWarp = 4;               // first of the eight epilogue warps
constexpr int kEpiWarps = 8;
constexpr int kTileA = kBM * 128;         // bytes of a weight tile: 128 rows of 128 bytes
constexpr int kMaxN = 256;                // rows of x per pass (128 for gate|up)
constexpr int kUnit = 4;                  // K steps whose scales are handed over together
constexpr int kScSlots = 3;               // ring of such units
constexpr int kMaxAcc = 8;
// Registers: 168 a thread at launch; the epilogue warpgroups hold up to 128 sums and two tiles of 32 columns a thread
// and take theirs from the first warpgroup: 128 * 88 + 256 * 208 = 64512 = the launch's 384 * 168.
constexpr int kLoadRegs = 88, kEpiRegs = 208;
constexpr int kMaxStages = 16;
constexpr int kTmemCols = 512;
constexpr int kRowMaps = 5;               // boxes of 16, 32, .., 256 rows of x
constexpr int kMaxSmem = 232448;          // 227 KB
constexpr int kMaxRed = 64 << 10;         // shared memory for partial sums of a split

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
    int Kb;                    // K steps (128 bytes of a row each)
    int Mb;                    // blocks of 128 output columns
    int NT;                    // rows of x per pass, at most
    int stages;
    int nacc;                  // accumulator slots in TMEM
    int acc_cols;              // TMEM columns of one half of a slot; also rows of x in a scale slot
    int prom;                  // K steps summed in TMEM before their sum is added to the f32 registers
    int vec;                   // whole rows of results start on 16-byte boundaries
};

struct Maps {
    CUtensorMap w;
    CUtensorMap x[kRowMaps];
};

// The items of this CTA (of its group of `split` CTAs, when items are split over K).
struct Items {
    const GroupedArgs& a;
    const int2* meta;          // (first row, rows) of each expert
    const int* pstart;         // first item of each expert; [E]: all items
    int it, step, e, mb, row0, nrows;
    __device__ Items(const GroupedArgs& args, const int2* m, const int* ps, int first, int by)
        : a(args), meta(m), pstart(ps), it(first - by), step(by), e(0)
    {
    }
    __device__ bool next()
    {
        it += step;
        if (it >= pstart[a.E]) return false;
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
        const int passes = (m.y + a.NT - 1) / a.NT;
        const int local = it - pstart[e];
        mb = local / passes;
        const int pass = local - mb * passes;
        const int size = ((m.y + passes - 1) / passes + 15) & ~15;     // passes of about equal size
        row0 = m.x + pass * size;
        nrows = min(size, m.y - pass * size);
        return true;
    }
};

// The K steps k0 .. k1 - 1 of one item after another, kUnit at a time.
struct Units {
    Items w;
    int k0, k1, kb;
    bool live;
    __device__ Units(const Items& items, int first, int last) : w(items), k0(first), k1(last), kb(first)
    {
        live = w.next();
    }
    __device__ void next()
    {
        if (live && (kb += kUnit) >= k1) {
            live = w.next();
            kb = k0;
        }
    }
};

__device__ __forceinline__ uint64_t pack2(float lo, float hi)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t a, uint64_t b)
{
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

__device__ __forceinline__ void add2(uint64_t& acc, uint64_t a)
{
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(a));
}

template <int OUT>
struct OutOf;
template <>
struct OutOf<MB_T_F32> {
    using T = float;
    static __device__ __forceinline__ T round(float v) { return v; }
};
template <>
struct OutOf<MB_T_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ T round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct OutOf<MB_T_F16> {
    using T = __half;
    static __device__ __forceinline__ T round(float v) { return __float2half_rn(v); }
};

// Results of 32 rows wait in shared memory as rows of 128 outputs, f32 ones in two halves of 16 rows.  The distance
// between rows keeps the fragments' stores (4 rows 2 apart x 8 outputs) on different banks.
__host__ __device__ constexpr int out_bytes(int out) { return out == MB_T_F32 ? 4 : out == MB_T_E4M3 ? 1 : 2; }
__host__ __device__ constexpr int tile_rows(int out) { return out == MB_T_F32 ? 16 : 32; }
__host__ __device__ constexpr int tile_pitch(int out) { return 128 * out_bytes(out) + 16; }

// Where scale n of 32 lies: a thread reads those of its columns 8 b + 2 i + e (i = lane % 4), b = 0, 1, as one vector.
__device__ __forceinline__ int scale_pos(int n) { return (n & ~15) + ((n >> 1) & 3) * 4 + ((n >> 3) & 1) * 2 + (n & 1); }

// What an epilogue warp keeps between items.
struct Epilogue {
    const GroupedArgs& a;
    unsigned* status;
    volatile int* abort_flag;
    uint32_t tl;               // TMEM address of the warp's lane quarter
    uint64_t *acc_full, *acc_empty, *sc_full, *sc_empty;
    const float* sc;
    uint64_t* red;
    uint64_t *red_full, *red_empty;
    float *amax, *tsc;
    uint8_t* tile;             // the set's rows of results
    int k0, k1, split, srank;
    uint32_t leader;
    int q, set, lane;
    Ring ac, scr;
    int sent, abuf;

    // One item with N chunks of 32 rows for this warp's set (a count known at compile time keeps the sums in
    // registers: with a test around each chunk a step took 3200 cycles at 256 rows, most of them moves).
    // sum[t][8 h + 2 b + s]: weight row 32 q + 16 h + 8 s + lane / 4, rows of x 8 b + 2 (lane % 4) + {0, 1} of tile t.
    template <int TYPE, bool DUAL, int OUT, int N>
    __device__ __forceinline__ void item(const Items& w)
    {
        constexpr bool FP8 = TYPE == MB_T_E4M3;
        constexpr int H = DUAL ? 2 : 1;
        constexpr int T = H * N;               // tiles of 32 columns: chunk t / H, half t % H
        const int scw = H * a.acc_cols;
        bool ok = true;
        uint64_t sum[T > 0 ? T : 1][16];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[t][j] = 0;
        for (int kb = k0; kb < k1; kb += a.prom) {
            const int us = (kb - k0) % kUnit;
            if (FP8 && us == 0) ok = mb_mbar_wait_spin(&sc_full[scr.slot], scr.full_parity(), status, abort_flag) && ok;
            ok = mb_mbar_wait_spin(&acc_full[ac.slot], ac.full_parity(), status, abort_flag) && ok;
            tc_after();
            if constexpr (T > 0) {
                float d[2][32];                // the next tile is on its way while this one is added
                const uint32_t from = tl + ac.slot * scw + 32 * set;
                const float* s0 = sc + (scr.slot * kUnit + us) * scw + 32 * set + 4 * (lane & 3);
                tc_ld32(from, d[0]);
                tc_wait_ld();
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    if (t + 1 < T) tc_ld32(from + ((t + 1) % H) * a.acc_cols + 64 * ((t + 1) / H), d[(t + 1) & 1]);
                    const float(&v)[32] = d[t & 1];
#pragma unroll
                    for (int bp = 0; bp < 2; ++bp) {
                        float4 s = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                        if (FP8)
                            s = *reinterpret_cast<const float4*>(s0 + (t % H) * a.acc_cols + 64 * (t / H) + 16 * bp);
#pragma unroll
                        for (int r = 0; r < 8; ++r) {      // b = 2 bp + r % 2, s = r / 2 % 2, h = r / 4
                            const int b = 2 * bp + (r & 1), j = 8 * (r >> 2) + 2 * b + ((r >> 1) & 1);
                            const uint64_t x = pack2(v[2 * j], v[2 * j + 1]);
                            if (FP8)
                                fma2(sum[t][j], x, r & 1 ? pack2(s.z, s.w) : pack2(s.x, s.y));
                            else
                                add2(sum[t][j], x);
                        }
                    }
                    if (t + 1 < T) tc_wait_ld();
                }
            }
            tc_before();
            __syncwarp();
            const bool unit_done = FP8 && (us == kUnit - 1 || kb + 1 == k1);
            if (lane == 0) {
                mb_mbar_arrive(&acc_empty[ac.slot]);
                if (unit_done) mb_mbar_arrive(&sc_empty[scr.slot]);
            }
            ac.next();
            if (unit_done) scr.next();
        }

        if (split > 1) {
            // NT <= 32: one chunk, one set.  Partial sums: [sender][half][h, b, s][128 threads] pairs.
            const int np = (w.nrows + 15) & ~15, nb = a.NT / 8;
            const int me = 32 * q + lane;
            if (srank > 0) {
                // the receiver has read the previous item's sums (the first wait passes at once)
                ok = mbar_wait_cluster(red_empty, (sent & 1) ^ 1, status, abort_flag) && ok;
                ++sent;
                if constexpr (N == 1) {
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const uint32_t to =
                            cluster_map(mb_smem_addr(red + ((srank - 1) * H + h) * 4 * nb * 128 + me), leader);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int b = (j >> 1) & 3;
                            if (8 * b < np && ok) cluster_st(to + (((j >> 3) * nb + b) * 2 + (j & 1)) * 1024, sum[h][j]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) cluster_arrive(cluster_map(mb_smem_addr(red_full), leader));
                return;
            }
            ok = mbar_wait_cluster(red_full, sent & 1, status, abort_flag) && ok;
            ++sent;
            if constexpr (N == 1) {
                for (int r = 0; r < split - 1; ++r)
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        const uint64_t* from = red + (r * H + h) * 4 * nb * 128 + me;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int b = (j >> 1) & 3;
                            if (8 * b < np) add2(sum[h][j], from[(((j >> 3) * nb + b) * 2 + (j & 1)) * 128]);
                        }
                    }
            }
            __syncwarp();
            if (lane == 0)
                for (int r = 1; r < split; ++r) cluster_arrive(cluster_map(mb_smem_addr(red_empty), leader + r));
        }

#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = 2 * i + set;
            const int n = w.nrows - 32 * c;                // rows of this chunk (32 or fewer are real)
            const int64_t row = (int64_t)w.row0 + 32 * c;
            float v[32];
#pragma unroll
            for (int j = 0; j < 16; ++j) unpack2(sum[H * i][j], v[2 * j], v[2 * j + 1]);
            if constexpr (DUAL) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float u0, u1;
                    unpack2(sum[H * i + 1][j], u0, u1);
                    v[2 * j] = __fdividef(v[2 * j], 1.0f + __expf(-v[2 * j])) * u0;
                    v[2 * j + 1] = __fdividef(v[2 * j + 1], 1.0f + __expf(-v[2 * j + 1])) * u1;
                }
            }
            if constexpr (OUT == MB_T_E4M3)
                encode(w.mb, v, row, n, ok);
            else
                store<OUT>(w.mb, v, row, n, ok);
        }
    }

    // The tile's rows to y, 128 outputs (fewer in the last block) from column 128 mb on: `rows` rows of out bytes each.
    template <int OUT>
    __device__ __forceinline__ void send(int mb, int64_t row, int rows, bool ok)
    {
        constexpr int R = tile_rows(OUT), B = out_bytes(OUT), pitch = tile_pitch(OUT);
        bulk_fence();
        mb_named_barrier(1 + set, 128);
        const int me = 32 * q + lane, bytes = min(kBM, a.O - mb * kBM) * B;
        uint8_t* dst = reinterpret_cast<uint8_t*>(a.y) + (row * a.ldy + (int64_t)mb * kBM) * B;
        if (a.vec && bytes % 16 == 0) {
            const int r = me / (128 / R);
            if (me % (128 / R) == 0 && r < rows && ok)
                bulk_s2g(dst + r * a.ldy * B, tile + r * pitch, bytes);
            bulk_commit();
        } else if (ok) {
            for (int r = q; r < min(rows, R); r += 4)
                for (int i = lane; i < bytes / B; i += 32)
                    if (B == 4)
                        reinterpret_cast<uint32_t*>(dst + r * a.ldy * B)[i] = reinterpret_cast<uint32_t*>(tile + r * pitch)[i];
                    else if (B == 2)
                        reinterpret_cast<uint16_t*>(dst + r * a.ldy * B)[i] = reinterpret_cast<uint16_t*>(tile + r * pitch)[i];
                    else
                        (dst + r * a.ldy)[i] = (tile + r * pitch)[i];
        }
    }

    // 32 rows of results (this thread's fragment of them), rounded to the output type.
    template <int OUT>
    __device__ __forceinline__ void store(int mb, const float (&v)[32], int64_t row, int n, bool ok)
    {
        constexpr int R = tile_rows(OUT), pitch = tile_pitch(OUT);
        using O = OutOf<OUT>;
#pragma unroll
        for (int p = 0; p < 32 / R; ++p) {
            if (p * R >= n) break;
            bulk_wait_read();
            mb_named_barrier(1 + set, 128);                // the tile's last rows have left
            uint8_t* to = tile + 2 * (lane & 3) * pitch + (32 * q + (lane >> 2)) * out_bytes(OUT);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int b = (j >> 1) & 3, w = 16 * (j >> 3) + 8 * (j & 1);
                if (8 * b / R == p) {
                    typename O::T* d = reinterpret_cast<typename O::T*>(to + (8 * b - p * R) * pitch) + w;
                    d[0] = O::round(v[2 * j]);
                    d[pitch / out_bytes(OUT)] = O::round(v[2 * j + 1]);
                }
            }
            send<OUT>(mb, row + p * R, n - p * R, ok);
        }
    }

    // 32 rows of results as e4m3 with a scale per row: each row's largest of the block's 128 columns (over a thread's
    // four, the eight lanes that share its rows, and the set's four warps), then the quotients.
    __device__ __forceinline__ void encode(int mb, const float (&v)[32], int64_t row, int n, bool ok)
    {
        constexpr int pitch = tile_pitch(MB_T_E4M3);
        const int o = mb * kBM + 32 * q + (lane >> 2);
        float m[8];                                        // index 2 b + e
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int b = (j >> 1) & 3;
            if (o + 16 * (j >> 3) + 8 * (j & 1) < a.O) {
                m[2 * b] = fmaxf(m[2 * b], fabsf(v[2 * j]));
                m[2 * b + 1] = fmaxf(m[2 * b + 1], fabsf(v[2 * j + 1]));
            }
        }
#pragma unroll
        for (int s = 16, h = 4; s >= 4; s >>= 1, h >>= 1) {
            const bool hi = lane & s;
#pragma unroll
            for (int i = 0; i < h; ++i) {
                const float send = hi ? m[i] : m[i + h], keep = hi ? m[i + h] : m[i];
                m[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, s));
            }
        }
        // this lane now has index lane / 4
        float* am = amax + ((set * 2 + abuf) * 4) * 32;
        abuf ^= 1;
        am[q * 32 + 8 * (lane >> 3) + 2 * (lane & 3) + ((lane >> 2) & 1)] = m[0];
        bulk_wait_read();
        mb_named_barrier(1 + set, 128);                    // also: the tile's last rows have left
        const Quotient qu(e4m3_scale(fmaxf(fmaxf(am[lane], am[32 + lane]), fmaxf(am[64 + lane], am[96 + lane]))));
        const bool fast = __all_sync(0xffffffffu, qu.fast);
        float* ts = tsc + (set * 4 + q) * 64;
        ts[lane] = qu.s;
        ts[32 + lane] = qu.r;
        if (q == 0 && lane < n && ok) a.qs[(row + lane) * a.qs_row + mb * a.qs_group] = qu.s;
        __syncwarp();
        uint8_t* to = tile + 2 * (lane & 3) * pitch + 32 * q + (lane >> 2);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float2 s = *reinterpret_cast<const float2*>(ts + 8 * b + 2 * (lane & 3));
            const float2 r = *reinterpret_cast<const float2*>(ts + 32 + 8 * b + 2 * (lane & 3));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 8 * (i >> 1) + 2 * b + (i & 1);
                const float x0 = v[2 * j], x1 = v[2 * j + 1];
                const uint32_t e = fast ? to_e4m3x2(quotient(x0, s.x, r.x), quotient(x1, s.y, r.y))
                                        : to_e4m3x2(__fdiv_rn(x0, s.x), __fdiv_rn(x1, s.y));
                uint8_t* d = to + 8 * b * pitch + 16 * (i >> 1) + 8 * (i & 1);
                d[0] = (uint8_t)e;
                d[pitch] = (uint8_t)(e >> 8);
            }
        }
        send<MB_T_E4M3>(mb, row, n, ok);
    }
};

template <int R>
__device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// OUT: the result type (gate|up: TYPE)
template <int TYPE, bool DUAL, int OUT>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_kernel(const __grid_constant__ GroupedArgs a, const __grid_constant__ Maps maps)
{
    constexpr bool FP8 = TYPE == MB_T_E4M3;
    constexpr int KS = FP8 ? 128 : 64;    // columns of a K step
    constexpr int H = DUAL ? 2 : 1;       // weight tiles of a step

    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = H * kTileA + a.NT * 128;
    const uint32_t csize = cluster_size();
    uint8_t* stage0 = smem;
    const int sets = a.NT > 32 ? 2 : 1;   // passes of 32 rows or fewer have one chunk: one set of epilogue warps
    const int scw = H * a.acc_cols;
    uint64_t* red = reinterpret_cast<uint64_t*>(stage0 + (size_t)a.stages * stage_bytes);   // [csize - 1][H][NT / 2][128]
    float* sc = reinterpret_cast<float*>(red + (csize - 1) * H * a.NT * 64);                // [kScSlots][kUnit][scw]
    float* amax = sc + (FP8 ? kScSlots * kUnit * scw : 0);             // [2 sets][2][4 quarters][32]
    float* tsc = amax + (OUT == MB_T_E4M3 ? 2 * 2 * 4 * 32 : 0);       // [8 warps][scale, 1 / scale][32]
    uint8_t* tiles = reinterpret_cast<uint8_t*>(tsc + (OUT == MB_T_E4M3 ? kEpiWarps * 64 : 0));   // [sets][rows][pitch]
    uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + sets * tile_rows(OUT) * tile_pitch(OUT));
    uint64_t* full = bars;
    uint64_t* empty = full + kMaxStages;
    uint64_t* acc_full = empty + kMaxStages;
    uint64_t* acc_empty = acc_full + kMaxAcc;
    uint64_t* sc_full = acc_empty + kMaxAcc;
    uint64_t* sc_empty = sc_full + kScSlots;
    uint64_t* red_full = sc_empty + kScSlots;
    uint64_t* red_empty = red_full + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(red_empty + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* wsum = reinterpret_cast<int*>(tmem_slot + 2);                 // [kThreadWarps] + split
    int2* meta = reinterpret_cast<int2*>(wsum + 16);                   // [E]
    int* pstart = reinterpret_cast<int*>(meta + a.E);                  // [E + 1]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned* const status = a.status ? a.status : &g_no_status;

    mb_pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            mb_mbar_init(&full[i], 1);
            mb_mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < a.nacc; ++i) {
            mb_mbar_init(&acc_full[i], 1);
            mb_mbar_init(&acc_empty[i], 4 * sets);
        }
        for (int i = 0; i < kScSlots; ++i) {
            mb_mbar_init(&sc_full[i], 1);
            mb_mbar_init(&sc_empty[i], 4 * sets);
        }
        *abort_flag = 0;
        tma_prefetch_map(&maps.w);
    }
    if (warp == 1) tc_alloc(tmem_slot, kTmemCols);
    mb_pdl_wait();

    // The experts' rows and the first item of each: an exclusive scan over the experts, a run of them per thread.
    {
        const int per = (a.E + kThreads - 1) / kThreads;
        const int e0 = threadIdx.x * per, e1 = min(a.E, e0 + per);
        int items = 0;
        for (int e = e0; e < e1; ++e) {
            int lo = 0, n = (int)a.P;
            if (a.offsets) {
                lo = a.offsets[e];
                const int hi = a.offsets[e + 1];
                n = hi - lo;
                if (lo < 0 || hi < lo || hi > a.P) {
                    atomicOr(status, MB_STATUS_BADARG);
                    lo = n = 0;
                }
            }
            meta[e] = make_int2(lo, n);
            pstart[e] = items;
            items += a.Mb * ((n + a.NT - 1) / a.NT);
        }
        int run = items;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += t;
        }
        if (lane == 31) wsum[warp] = run;
        __syncthreads();
        int before = run - items, total = 0;
        for (int w = 0; w < kThreadWarps; ++w) {
            const int s = wsum[w];
            if (w < warp) before += s;
            total += s;
        }
        for (int e = e0; e < e1; ++e) pstart[e] += before;
        if (threadIdx.x == 0) {
            pstart[a.E] = total;
            // How many CTAs share an item: the split whose longest CTA has the fewest K steps, two more for each
            // item that is split (the partial sums' way to the first CTA).
            int best = 0x7fffffff, split = 1;
            for (int s = 1; s <= (int)csize && s <= a.Kb; s <<= 1) {
                const int groups = gridDim.x / s;
                const int64_t c = (int64_t)((total + groups - 1) / groups) * ((a.Kb + s - 1) / s + (s > 1 ? 2 : 0));
                if (c < best) {
                    best = (int)c;
                    split = s;
                }
            }
            wsum[15] = split;
            mb_mbar_init(red_full, 4 * max(split - 1, 1));  // a split needs NT <= 32: one set
            mb_mbar_init(red_empty, 4);
            mb_fence_mbar_init();
        }
    }
    tc_before();
    __syncthreads();
    if (csize > 1) cluster_sync();        // the other CTAs' barriers exist
    tc_after();

    const uint32_t tmem = *tmem_slot;
    const int split = wsum[15];
    const int srank = (int)blockIdx.x % split;                          // rank among the CTAs of an item
    const int k0 = (int)((int64_t)a.Kb * srank / split), k1 = (int)((int64_t)a.Kb * (srank + 1) / split);
    const uint32_t leader = cluster_rank() - srank;                     // cluster rank of the item's first CTA
    Items w(a, meta, pstart, blockIdx.x / split, gridDim.x / split);

    if (warp < kEpiWarp) setmaxnreg_dec<kLoadRegs>();
    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        Ring st(a.stages);
        bool ok = true;
        int issued = 0;
        while (ok && w.next()) {
            const int r16 = (w.nrows + 15) >> 4;
            // lanes 0, 1: weight tiles; lane 2 + b: a box of 16 << b rows, the larger boxes first
            const int b = lane - 2;
            const bool box = b >= 0 && b < kRowMaps && ((r16 >> b) & 1);
            const int brow = b >= 0 && b < kRowMaps ? ((r16 >> (b + 1)) << (b + 1)) * 16 : 0;
            for (int kb = k0; kb < k1; ++kb, st.next()) {
                ok = __all_sync(0xffffffffu, mb_mbar_wait_spin(&empty[st.slot], st.empty_parity(), status, abort_flag));
                if (!ok) break;
                uint8_t* dst = stage0 + (size_t)st.slot * stage_bytes;
                if (lane == 0) mb_mbar_arrive_expect_tx(&full[st.slot], H * kTileA + r16 * 16 * 128);
                __syncwarp();
                if (lane < H)
                    tma_load3(dst + lane * kTileA, &maps.w, kb * KS, lane * a.O + w.mb * kBM, w.e, &full[st.slot]);
                else if (box)
                    tma_load2(dst + H * kTileA + brow * 128, &maps.x[b], kb * KS, w.row0 + brow, &full[st.slot]);
                ++issued;
            }
        }
        if (!ok) {   // wait (bounded) for the copies still in flight before the CTA may end
            for (int i = 0; i < min(issued, a.stages); ++i) {
                if (--st.slot < 0) {
                    st.slot = a.stages - 1;
                    st.phase ^= 1;
                }
                for (int n = 0; n < 100000 && !mb_mbar_try_wait(&full[st.slot], st.full_parity()); ++n) {
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ tensor cores
        if (elect_one()) {
            Ring st(a.stages), ac(a.nacc);
            bool ok = true;
            // D f32; A and B both K-major: e4m3 / f16 are format 0, bf16 is 1
            const uint32_t fmt = TYPE == MB_T_BF16 ? (1u << 7) | (1u << 10) : 0u;
            const uint64_t desc0 = tc_desc_sw128(mb_smem_addr(stage0));
            while (ok && w.next()) {
                const int n16 = (w.nrows + 15) & ~15;
                const uint32_t idesc = (1u << 4) | fmt | ((uint32_t)(n16 >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
                int part = 0;                              // K steps already in the accumulator
                for (int kb = k0; kb < k1; ++kb, st.next()) {
                    if (part == 0)
                        ok = mb_mbar_wait_spin(&acc_empty[ac.slot], ac.empty_parity(), status, abort_flag);
                    ok = ok && mb_mbar_wait_spin(&full[st.slot], st.full_parity(), status, abort_flag);
                    if (!ok) break;
                    tc_after();
                    const uint64_t da = desc0 + (uint64_t)((st.slot * stage_bytes) >> 4);
                    const uint64_t db = da + (H * kTileA >> 4);
                    const uint32_t d = tmem + ac.slot * scw;
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tc_mma_ss<FP8>(d + h * a.acc_cols, da + (h * kTileA >> 4) + 2 * j, db + 2 * j, idesc,
                                           (j > 0 || part > 0) ? 1u : 0u);
                    tc_commit(&empty[st.slot]);
                    if (++part == a.prom || kb + 1 == k1) {
                        tc_commit(&acc_full[ac.slot]);
                        ac.next();
                        part = 0;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp < kEpiWarp) {
        // ------------------------------------------------------------------ scales (steps in turn between two warps)
        if (FP8) {
            // Each warp takes every second unit.  A lane loads kUnit groups of its rows at once: the scales come from L2 or
            // HBM, and four groups share that latency and the hand-over.
            constexpr int NL = DUAL ? 4 : 8;               // rows per lane
            const int Ob = (a.O + kScaleBlock - 1) / kScaleBlock;
            Units un(w, k0, k1);
            if (warp == 3) un.next();
            Ring slot(kScSlots);
            if (warp == 3) slot.next();
            while (un.live) {
                const int m = min(kUnit, k1 - un.kb);
                const float* wsp = a.ws + ((int64_t)un.w.e * H * Ob + un.w.mb) * a.Kb + un.kb;
                const float* xsp = a.xs + ((int64_t)un.w.row0 + lane) * a.xs_row + (int64_t)un.kb * a.xs_group;
                float v[NL][kUnit], w0[kUnit], w1[kUnit];
#pragma unroll
                for (int s = 0; s < kUnit; ++s) {
                    w0[s] = s < m ? wsp[s] : 0.0f;
                    if (DUAL) w1[s] = s < m ? wsp[(int64_t)Ob * a.Kb + s] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    const bool real = lane + 32 * i < un.w.nrows;
#pragma unroll
                    for (int s = 0; s < kUnit; ++s)
                        v[i][s] = real && s < m ? xsp[(int64_t)(32 * i) * a.xs_row + s * a.xs_group] : 0.0f;
                }
                if (!__all_sync(0xffffffffu, mb_mbar_wait_spin(&sc_empty[slot.slot], slot.empty_parity(), status,
                                                              abort_flag)))
                    break;
                float* dst = sc + slot.slot * kUnit * scw + scale_pos(lane);
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    if (32 * i >= un.w.nrows) break;
#pragma unroll
                    for (int s = 0; s < kUnit; ++s) {
                        dst[s * scw + 32 * i] = v[i][s] * w0[s];
                        if (DUAL) dst[s * scw + a.acc_cols + 32 * i] = v[i][s] * w1[s];
                    }
                }
                __syncwarp();
                if (lane == 0) mb_mbar_arrive(&sc_full[slot.slot]);
                un.next();
                un.next();
                slot.next();
                slot.next();
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        setmaxnreg_inc<kEpiRegs>();
        const int set = (warp - kEpiWarp) >> 2;
        if (set < sets) {
            Epilogue ep{a, status, abort_flag, tmem + ((uint32_t)(32 * (warp & 3)) << 16), acc_full, acc_empty,
                        sc_full, sc_empty, sc, red, red_full, red_empty, amax, tsc,
                        tiles + set * tile_rows(OUT) * tile_pitch(OUT), k0, k1, split, srank, leader,
                        warp & 3, set, lane, Ring(a.nacc), Ring(kScSlots), 0, 0};
            while (w.next()) {
                const int nch = (w.nrows + 31) >> 5;       // chunks of 32 rows; this set takes set, set + 2, ..
                const int mine = (nch - set + 1) >> 1;
                if (mine == 0)
                    ep.item<TYPE, DUAL, OUT, 0>(w);
                else if (mine == 1)
                    ep.item<TYPE, DUAL, OUT, 1>(w);
                else if (mine == 2)
                    ep.item<TYPE, DUAL, OUT, 2>(w);
                else if constexpr (!DUAL) {
                    if (mine == 3)
                        ep.item<TYPE, DUAL, OUT, 3>(w);
                    else
                        ep.item<TYPE, DUAL, OUT, 4>(w);
                }
            }
            bulk_wait();
        }
    }

    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 1) tc_dealloc(tmem, kTmemCols);
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


int make_maps(const GroupedArgs& a, int type, int halves, Maps* m, const char* what)
{
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return mb_fail(MB_ECUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
    const cuuint64_t b = (cuuint64_t)elem_bytes(type);
    const cuuint32_t inner = (cuuint32_t)(128 / b), one[3] = {1, 1, 1};
    const cuuint64_t wd[3] = {(cuuint64_t)a.K, (cuuint64_t)a.O * halves, (cuuint64_t)a.E};
    const cuuint64_t wst[2] = {(cuuint64_t)a.ldw * b,
                               (cuuint64_t)(a.E > 1 ? a.w_expert : (int64_t)a.O * halves * a.ldw) * b};
    const cuuint32_t wbox[3] = {inner, kBM, 1};
    CUresult r = fn(&m->w, map_type(type), 3, const_cast<void*>(a.w), wd, wst, wbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    const cuuint64_t xd[2] = {(cuuint64_t)a.K, (cuuint64_t)a.P};
    const cuuint64_t xst[1] = {(cuuint64_t)a.ldx * b};
    for (int i = 0; i < kRowMaps && (16 << i) <= a.NT && r == CUDA_SUCCESS; ++i) {
        const cuuint32_t xbox[2] = {inner, (cuuint32_t)(16 << i)};
        r = fn(&m->x[i], map_type(type), 2, const_cast<void*>(a.x), xd, xst, xbox, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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

template <int TYPE, bool DUAL, int OUT>
int launch(GroupedArgs a, const char* what, cudaStream_t st)
{
    constexpr bool FP8 = TYPE == MB_T_E4M3;
    constexpr int H = DUAL ? 2 : 1;
    const int sms = mb_num_sms();
    a.Kb = (a.K + (FP8 ? 127 : 63)) / (FP8 ? 128 : 64);
    a.Mb = (a.O + kBM - 1) / kBM;
    const int maxn = DUAL ? kMaxN / 2 : kMaxN;
    const int64_t active = std::min<int64_t>(a.E, a.P);          // experts with rows, at most
    if (a.offsets) {
        a.NT = pow2_at_least((a.P * 3 / 2 + a.E - 1) / a.E, 16, maxn);
    } else {
        a.NT = pow2_at_least(a.P, 16, maxn);
        while (a.NT > 32 && a.Mb * ((a.P + a.NT - 1) / a.NT) < sms) a.NT >>= 1;
    }
    const int64_t items = (int64_t)a.Mb * (active + a.P / a.NT);   // an upper bound
    MB_REQUIRE(items < (1ll << 30), "%s: %lld work items", what, (long long)items);
    int cluster = 1;
    if (a.NT <= 32 && a.Mb * active < 4 * sms)
        while (cluster < 8 && cluster * 2 <= a.Kb && (2 * cluster - 1) * H * a.NT * 512 <= kMaxRed &&
               a.Mb * active * cluster < 4 * sms)
            cluster *= 2;
    a.acc_cols = std::max(32, a.NT);
    a.nacc = std::min(kMaxAcc, kTmemCols / (H * a.acc_cols));
    a.prom = FP8 ? 1 : OUT == MB_T_F32 ? 4 : a.Kb;
    a.vec = ((uintptr_t)a.y & 15) == 0 && a.ldy * out_bytes(OUT) % 16 == 0;
    const int stage = H * kTileA + a.NT * 128;
    const int scales = FP8 ? kScSlots * kUnit * H * a.acc_cols * 4 : 0;
    const int encode = OUT == MB_T_E4M3 ? 2 * 2 * 4 * 32 * 4 + kEpiWarps * 64 * 4 : 0;
    const int tiles = (a.NT > 32 ? 2 : 1) * tile_rows(OUT) * tile_pitch(OUT);
    const int fixed = 1024 + (cluster - 1) * H * a.NT * 512 + scales + encode + tiles +
                      (2 * kMaxStages + 2 * kMaxAcc + 2 * kScSlots + 2) * 8 + 8 + 64 + a.E * 8 + (a.E + 1) * 4 + 16;
    a.stages = std::min(kMaxStages, (kMaxSmem - fixed) / stage);
    const int smem = fixed + a.stages * stage;

    auto kern = grouped_kernel<TYPE, DUAL, OUT>;
    static thread_local uint64_t ready = 0;                        // devices whose attribute is set
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(ready >> (dev & 63) & 1)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return mb_fail(MB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
        ready |= 1ull << (dev & 63);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = kThreads;
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
    int ctas = sms;
    if (cluster > 1) {
        // clusters that fit at the same time: a CTA takes an SM, and a cluster stays within one GPC
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
    const int rc = make_maps(a, TYPE, H, &maps, what);
    if (rc) return rc;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, maps);
    if (e != cudaSuccess) return mb_fail(MB_ECUDA, "%s: %s", what, cudaGetErrorString(e));
    return MB_OK;
}

template <int TYPE>
int launch_as(const GroupedArgs& a, int y_type, const char* what, cudaStream_t st)
{
    if (y_type == MB_T_F32) return launch<TYPE, false, MB_T_F32>(a, what, st);
    if (y_type == MB_T_BF16) return launch<TYPE, false, MB_T_BF16>(a, what, st);
    return launch<TYPE, false, MB_T_F16>(a, what, st);
}

int matmul(GroupedArgs a, int type, int y_type, const char* what, void* stream)
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

extern "C" int mb_grouped_matmul_t(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                   int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                   const float* ws, int E, int O, int K, const int32_t* offsets, void* y, int y_type,
                                   int64_t ldy, unsigned* status, void* stream)
{
    MB_REQUIRE(offsets || P == 0, "mb_grouped_matmul_t: null pointer");
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, O, K,
                        offsets, y, ldy, nullptr, 0, 0, status};
    return matmul(a, type, y_type, "mb_grouped_matmul_t", stream);
}

extern "C" int mb_matmul_t_e4m3(const void* x, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_group,
                                int64_t n, const void* w, int64_t ldw, const float* ws, int O, int K, void* y,
                                int y_type, int64_t ldy, unsigned* status, void* stream)
{
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, n, w, 0, ldw, ws, 1, O, K,
                        nullptr, y, ldy, nullptr, 0, 0, status};
    return matmul(a, MB_T_E4M3, y_type, "mb_matmul_t_e4m3", stream);
}

extern "C" int mb_grouped_swiglu_t(const void* x, int type, int64_t ldx, const float* xs, int64_t xs_row,
                                   int64_t xs_group, int64_t P, const void* w, int64_t w_expert, int64_t ldw,
                                   const float* ws, int E, int I, int K, const int32_t* offsets, void* q, int64_t ldq,
                                   float* qs, int64_t qs_row, int64_t qs_group, unsigned* status, void* stream)
{
    const char* what = "mb_grouped_swiglu_t";
    MB_REQUIRE(offsets || P == 0, "%s: null pointer", what);
    const GroupedArgs a{x, ldx, xs, xs_row, xs_group, P, w, w_expert, ldw, ws, E, I, K,
                        offsets, q, ldq, qs, qs_row, qs_group, status};
    int rc = check_args(a, type, 2, what);
    if (rc || P == 0) return rc;
    MB_REQUIRE(type != MB_T_E4M3 || qs, "%s: e4m3 results need their scales", what);
    const cudaStream_t st = mb_stream(stream);
    if (type == MB_T_E4M3) return launch<MB_T_E4M3, true, MB_T_E4M3>(a, what, st);
    if (type == MB_T_BF16) return launch<MB_T_BF16, true, MB_T_BF16>(a, what, st);
    return launch<MB_T_F16, true, MB_T_F16>(a, what, st);
}
