// Operand rows: the rows of x picked by index, in the form the float experts'
// products read (e4m3 with one f32 scale per 128 columns, bf16 or f16).
//
// s = max|group| / 448 (448 is e4m3's largest value; 1 for a group of zeros),
// q = e4m3(x / s), both quotients and the cast rounded to nearest even, so the
// largest value of every group maps to +-448 and nothing saturates.
//
// A warp takes four groups of a row (512 columns): lane l holds columns 4l .. 4l+3 of each, loaded at once; the four
// maxima are reduced together, and each group's scale is worked out by the eight lanes that end with its maximum.
//
// Two kernels.  operand_rows_kernel makes each row of the result from its row of x; e4m3 rows are bound by instructions
// (about 200 a warp) when tokens have many picks, since every pick of a token repeats the work.  spread_rows_kernel, for
// e4m3, makes each row of x once, into shared memory, looks through `rows` for its picks and copies the row to them.
// Looking costs n * 4 bytes per sixteen rows of x, which pays for long rows.  us in graphs, made once / for each pick, from
// f32: 32768 rows of 2048 from 4096 30.0 / 46.2 (3.4 TB/s), 18944 from 2368 16.7 / 25.7, 9472 from 2368 10.4 / 13.9.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "mb_common.cuh"
#include "mb_float.cuh"

namespace {

constexpr int kGroups = 4;                // groups of a warp
constexpr int kRowsPerBlock = 8;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p)
{
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __half* p)
{
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Columns c0 + g * 128 .. + 3 of a row of x, g < kGroups (zeros past d, and where !ok).
template <typename SRC, bool VEC>
__device__ __forceinline__ void load_groups(float (&v)[kGroups][4], const SRC* from, int c0, int d, bool ok)
{
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int c = c0 + g * kScaleBlock;
        if (VEC) {
            const float4 t = ok && c < d ? load4(from + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v[g][0] = t.x, v[g][1] = t.y, v[g][2] = t.z, v[g][3] = t.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[g][i] = ok && c + i < d ? static_cast<float>(from[c + i]) : 0.0f;
        }
    }
}

// Each group's four values as e4m3 bytes; returns the scale of group lane / 8.
__device__ __forceinline__ float encode_groups(const float (&v)[kGroups][4], uint32_t (&u)[kGroups], int lane)
{
    // the groups' maxima: each lane keeps one group in the first two exchanges (lane / 8), then eight lanes share it
    float m[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
        m[g] = fmaxf(fmaxf(fabsf(v[g][0]), fabsf(v[g][1])), fmaxf(fabsf(v[g][2]), fabsf(v[g][3])));
#pragma unroll
    for (int o = 16, h = 2; h; o >>= 1, h >>= 1) {
        const bool hi = lane & o;
#pragma unroll
        for (int i = 0; i < h; ++i) {
            const float send = hi ? m[i] : m[i + h], keep = hi ? m[i + h] : m[i];
            m[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, o));
        }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
    const Quotient mine(e4m3_scale(m[0]));
    const bool fast = __all_sync(0xffffffffu, mine.fast);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const float s = __shfl_sync(0xffffffffu, mine.s, 8 * g), r = __shfl_sync(0xffffffffu, mine.r, 8 * g);
        float t[4] = {v[g][0], v[g][1], v[g][2], v[g][3]};
        if (fast) {
            quotient4(t, s, r);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = __fdiv_rn(t[i], s);
        }
        u[g] = to_e4m3x2(t[0], t[1]) | to_e4m3x2(t[2], t[3]) << 16;
    }
    return mine.s;
}

template <int TYPE>
__device__ __forceinline__ uint2 round4(const float (&v)[4])
{
    if (TYPE == MB_T_F16) return make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]));
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

struct RowsArgs {
    const void* x;
    int64_t ldx, n_src;
    const int32_t* rows;
    int64_t n;
    int d;
    void* q;
    int64_t ldq;
    float* scales;
    int64_t s_row, s_group;
    const int32_t *first, *last;           // null: every row
    unsigned* status;
};

// VEC: four columns at a time are aligned in x and q, and d is a multiple of 4.
template <typename SRC, int TYPE, bool VEC>
__global__ void operand_rows_kernel(const __grid_constant__ RowsArgs a)
{
    const SRC* __restrict__ x = reinterpret_cast<const SRC*>(a.x);
    const int32_t* __restrict__ rows = a.rows;
    void* __restrict__ q = a.q;
    float* __restrict__ scales = a.scales;
    unsigned* const status = a.status;
    const int64_t ldx = a.ldx, n_src = a.n_src, n = a.n, ldq = a.ldq, s_row = a.s_row, s_group = a.s_group;
    const int d = a.d;
    mb_pdl_trigger();
    mb_pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t p = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 5);
    if (p >= n || (a.first && (p < *a.first || p >= *a.last))) return;
    const int64_t src = rows ? rows[p] : p;
    const bool ok = src >= 0 && src < n_src;
    if (!ok && blockIdx.y == 0 && lane == 0 && status) atomicOr(status, MB_STATUS_BADARG);
    const int g0 = blockIdx.y * kGroups, c0 = g0 * kScaleBlock + 4 * lane;
    float v[kGroups][4];
    load_groups<SRC, VEC>(v, x + src * ldx, c0, d, ok);
    if constexpr (TYPE == MB_T_E4M3) {
        uint32_t u[kGroups];
        const float s = encode_groups(v, u, lane);
        if ((lane & 7) == 0 && (g0 + lane / 8) * kScaleBlock < d) scales[p * s_row + (g0 + lane / 8) * s_group] = s;
        uint8_t* dst = reinterpret_cast<uint8_t*>(q) + p * ldq;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int c = c0 + g * kScaleBlock;
            if (VEC) {
                if (c < d) *reinterpret_cast<uint32_t*>(dst + c) = u[g];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < d) dst[c + i] = (uint8_t)(u[g] >> (8 * i));
            }
        }
    } else {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int c = c0 + g * kScaleBlock;
            if (VEC) {
                if (c < d)
                    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(q) + p * ldq + c) = round4<TYPE>(v[g]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < d) store_out<TYPE>(q, p * ldq + c + i, v[g][i]);
            }
        }
    }
}

constexpr int kSpreadRows = 16;           // rows of x of a block, one per warp
constexpr int kSpreadThreads = 32 * kSpreadRows;
constexpr int kSegment = 4 * kSpreadThreads;   // picks looked through at a time
constexpr int kSpreadSmem = 88 << 10;     // for the rows, at most: two blocks per SM

// Sixteen rows of x, each put into e4m3 form once and copied to its picks.  Block 0 takes the picks of no row of x.
// Needs 16 bytes at a time to be aligned in q, four columns in x, and d a multiple of 16.
template <typename SRC>
__global__ void __launch_bounds__(kSpreadThreads) spread_rows_kernel(const SRC* __restrict__ x, int64_t ldx, int n_src,
                                                          const int32_t* __restrict__ rows, int n, int d,
                                                          uint8_t* __restrict__ q, int64_t ldq,
                                                          float* __restrict__ scales, int64_t s_row, int64_t s_group,
                                                          unsigned* status)
{
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint16_t found[kSegment], slots[kSegment];
    __shared__ int count;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ng = (d + kScaleBlock - 1) / kScaleBlock;
    float* sc = reinterpret_cast<float*>(smem + kSpreadRows * d);      // [kSpreadRows][ng]
    const int r0 = blockIdx.x * kSpreadRows;
    mb_pdl_trigger();
    mb_pdl_wait();

    int idx[kSegment / kSpreadThreads];                    // the next segment, on its way
    const int none = blockIdx.x == 0 ? kSpreadRows : 0;    // a row of x that is not this block's (there are more than 16)
    auto load = [&](int64_t base) {
#pragma unroll
        for (int j = 0; j < kSegment / kSpreadThreads; ++j) {
            const int64_t p = base + kSpreadThreads * j + threadIdx.x;
            idx[j] = p < n ? rows[p] : none;
        }
    };
    load(0);
    if (r0 + warp < n_src) {
        const SRC* from = x + (int64_t)(r0 + warp) * ldx;
        uint8_t* row = smem + warp * d;
        for (int g0 = 0; g0 < ng; g0 += kGroups) {
            const int c0 = g0 * kScaleBlock + 4 * lane;
            float v[kGroups][4];
            load_groups<SRC, true>(v, from, c0, d, true);
            uint32_t u[kGroups];
            const float s = encode_groups(v, u, lane);
            if ((lane & 7) == 0 && g0 + lane / 8 < ng) sc[warp * ng + g0 + lane / 8] = s;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int c = c0 + g * kScaleBlock;
                if (c < d) *reinterpret_cast<uint32_t*>(row + c) = u[g];
            }
        }
    }
    const unsigned mine = min(kSpreadRows, n_src - r0);
    for (int64_t base = 0; base < n; base += kSegment) {
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSegment / kSpreadThreads; ++j) {
            unsigned slot = (unsigned)idx[j] - (unsigned)r0;
            if (blockIdx.x == 0 && (unsigned)idx[j] >= (unsigned)n_src) slot = kSpreadRows;
            if (slot < mine || (blockIdx.x == 0 && slot == kSpreadRows && idx[j] != kSpreadRows)) {
                const int k = atomicAdd(&count, 1);        // (their order varies; every pick is one row's copy)
                found[k] = (uint16_t)(kSpreadThreads * j + threadIdx.x);
                slots[k] = (uint16_t)slot;
            }
        }
        __syncthreads();
        const int c = count;
        if (base + kSegment < n) load(base + kSegment);
        for (int k = warp; k < c; k += kSpreadRows) {
            const int slot = slots[k];
            const int64_t p = base + found[k];
            const bool real = slot < kSpreadRows;
            if (!real && lane == 0 && status) atomicOr(status, MB_STATUS_BADARG);
            uint8_t* dst = q + p * ldq;
            for (int i = 16 * lane; i < d; i += 512)
                *reinterpret_cast<uint4*>(dst + i) =
                    real ? *reinterpret_cast<const uint4*>(smem + slot * d + i) : make_uint4(0u, 0u, 0u, 0u);
            for (int g = lane; g < ng; g += 32) scales[p * s_row + g * s_group] = real ? sc[slot * ng + g] : 1.0f;
        }
        __syncthreads();
    }
}

template <typename SRC, int TYPE>
int launch(const SRC* x, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n, int d, void* q, int64_t ldq,
           float* scales, int64_t s_row, int64_t s_group, const int32_t* first, const int32_t* last, unsigned* status,
           cudaStream_t st)
{
    constexpr int B = TYPE == MB_T_E4M3 ? 1 : 2;
    const bool vec = d % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && (uintptr_t)x % (4 * sizeof(SRC)) == 0 &&
                     (uintptr_t)q % (4 * B) == 0;
    // Made once: e4m3, from four picks a row on, with a block of rows for every SM (16384 from 2048 rows of 2048: 23.7 us,
    // made for each pick 22.5; 9600 from 1200: 19.1 and 13.2), and at most four rows of x a column, since looking through
    // the picks (4 n bytes for each 16 rows) has to stay below the work it saves (us, once / each: 2368 rows x 8 of 1024
    // columns 13.0 / 13.9, of 512 11.7 / 8.0; 4096 x 8 of 1024 22.0 / 22.5, of 512 19.9 / 12.3; 8192 x 8 of 2048 83.9 /
    // 92.7, of 1024 71.3 / 46.5).  Rows of 16 bits cost little to make again, and the copies lose at every size (4096 x 8 of
    // 2048 columns 34.8 / 29.9, from bf16 41.5 / 25.3).  A slice of the experts has a part of the picks and is
    // made for each (its bounds in the other kernel cost every call 1.1 of 29.4 us at 32768 from 4096).
    if constexpr (TYPE == MB_T_E4M3) {
        const int ng = (d + kScaleBlock - 1) / kScaleBlock;
        const int64_t smem = (int64_t)kSpreadRows * (d + ng * 4);
        if (rows && !first && vec && n >= 4 * n_src && n_src >= kSpreadRows * mb_num_sms() && n_src <= 4 * (int64_t)d &&
            smem <= kSpreadSmem && d % 16 == 0 && ldq % 16 == 0 && (uintptr_t)q % 16 == 0) {
            static thread_local uint64_t ready = 0;        // devices whose attribute is set
            int dev = 0;
            cudaGetDevice(&dev);
            cudaError_t e = cudaSuccess;
            if (!(ready >> (dev & 63) & 1))
                e = cudaFuncSetAttribute(spread_rows_kernel<SRC>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpreadSmem);
            if (e == cudaSuccess) {
                ready |= 1ull << (dev & 63);
                e = mb_launch_pdl(spread_rows_kernel<SRC>, dim3((unsigned)((n_src + kSpreadRows - 1) / kSpreadRows)),
                                  dim3(kSpreadThreads), (size_t)smem, st, x, ldx, (int)n_src, rows, (int)n, d, (uint8_t*)q,
                                  ldq, scales, s_row, s_group, status);
            }
            if (e != cudaSuccess) return mb_fail(MB_ECUDA, "mb_operand_rows: %s", cudaGetErrorString(e));
            return MB_OK;
        }
    }
    const int cols = kGroups * kScaleBlock;
    const dim3 grid((unsigned)((n + kRowsPerBlock - 1) / kRowsPerBlock), (unsigned)((d + cols - 1) / cols));
    const RowsArgs a{x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, first, last, status};
    const cudaError_t e = mb_launch_pdl(vec ? operand_rows_kernel<SRC, TYPE, true> : operand_rows_kernel<SRC, TYPE, false>,
                                        grid, dim3(32 * kRowsPerBlock), 0, st, a);
    if (e != cudaSuccess) return mb_fail(MB_ECUDA, "mb_operand_rows: %s", cudaGetErrorString(e));
    return MB_OK;
}

template <typename SRC>
int launch_as(const SRC* x, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n, int d, int type, void* q,
              int64_t ldq, float* scales, int64_t s_row, int64_t s_group, const int32_t* first, const int32_t* last,
              unsigned* status, cudaStream_t st)
{
    if (type == MB_T_E4M3)
        return launch<SRC, MB_T_E4M3>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, first, last, status, st);
    if (type == MB_T_BF16)
        return launch<SRC, MB_T_BF16>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, first, last, status, st);
    return launch<SRC, MB_T_F16>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, first, last, status, st);
}

}  // namespace

extern "C" int mb_operand_rows_slice(const void* x, int x_type, int64_t ldx, int64_t n_src, const int32_t* rows,
                                     int64_t n, int d, int type, void* q, int64_t ldq, float* scales, int64_t s_row,
                                     int64_t s_group, const int32_t* first, const int32_t* last, unsigned* status,
                                     void* stream)
{
    MB_REQUIRE(x_type == MB_T_F32 || x_type == MB_T_BF16 || x_type == MB_T_F16, "mb_operand_rows: x type %d", x_type);
    MB_REQUIRE(type == MB_T_E4M3 || type == MB_T_BF16 || type == MB_T_F16, "mb_operand_rows: operand type %d", type);
    MB_REQUIRE(n >= 0 && n < (1ll << 31) && n_src >= 0 && d > 0 && d <= (1 << 24), "mb_operand_rows: n=%lld n_src=%lld d=%d",
               (long long)n, (long long)n_src, d);
    MB_REQUIRE(rows || n <= n_src, "mb_operand_rows: %lld rows of %lld", (long long)n, (long long)n_src);
    MB_REQUIRE(!first == !last, "mb_operand_rows: first without last");
    MB_REQUIRE(ldx >= d && ldq >= d, "mb_operand_rows: rows closer (%lld, %lld) than their width %d", (long long)ldx,
               (long long)ldq, d);
    if (n == 0) return MB_OK;
    MB_REQUIRE(q && (x || n_src == 0) && (type != MB_T_E4M3 || scales), "mb_operand_rows: null pointer");
    const cudaStream_t st = mb_stream(stream);
    if (x_type == MB_T_F32)
        return launch_as((const float*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, first, last, status,
                         st);
    if (x_type == MB_T_BF16)
        return launch_as((const __nv_bfloat16*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, first, last,
                         status, st);
    return launch_as((const __half*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, first, last, status,
                     st);
}

extern "C" int mb_operand_rows(const void* x, int x_type, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n,
                               int d, int type, void* q, int64_t ldq, float* scales, int64_t s_row, int64_t s_group,
                               unsigned* status, void* stream)
{
    return mb_operand_rows_slice(x, x_type, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, nullptr, nullptr,
                                 status, stream);
}
