// Operand rows: the rows of x picked by index, in the form the float experts'
// products read (e4m3 with one f32 scale per 128 columns, bf16 or f16).
//
// s = max|group| / 448 (448 is e4m3's largest value; 1 for a group of zeros),
// q = e4m3(x / s), both quotients and the cast rounded to nearest even, so the
// largest value of every group maps to +-448 and nothing saturates.
//
// A warp takes four groups of a row (512 columns): lane l holds columns 4l .. 4l+3 of each, loaded at once; the four
// maxima are reduced together, and each group's scale is worked out by the eight lanes that end with its maximum.  Bound by HBM (x in once, the rows out) and, with several picks a token, by reading
// x as often from L2.
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

// VEC: four columns at a time are aligned in x and q, and d is a multiple of 4.
template <typename SRC, int TYPE, bool VEC>
__global__ void operand_rows_kernel(const SRC* __restrict__ x, int64_t ldx, int64_t n_src,
                                    const int32_t* __restrict__ rows, int64_t n, int d, void* __restrict__ q,
                                    int64_t ldq, float* __restrict__ scales, int64_t s_row, int64_t s_group,
                                    unsigned* status)
{
    mb_pdl_trigger();
    mb_pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t p = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 5);
    if (p >= n) return;
    const int64_t src = rows ? rows[p] : p;
    const bool ok = src >= 0 && src < n_src;
    if (!ok && blockIdx.y == 0 && lane == 0 && status) atomicOr(status, MB_STATUS_BADARG);
    const int g0 = blockIdx.y * kGroups, c0 = g0 * kScaleBlock + 4 * lane;
    const SRC* from = x + src * ldx;
    float v[kGroups][4];
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
    if constexpr (TYPE != MB_T_E4M3) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int c = c0 + g * kScaleBlock;
            if (VEC) {
                uint2 u;
                if (TYPE == MB_T_BF16) {
                    const __nv_bfloat162 a = __floats2bfloat162_rn(v[g][0], v[g][1]);
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[g][2], v[g][3]);
                    u = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                } else {
                    u = make_uint2(pack_f16(v[g][0], v[g][1]), pack_f16(v[g][2], v[g][3]));
                }
                if (c < d) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(q) + p * ldq + c) = u;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < d) store_out<TYPE>(q, p * ldq + c + i, v[g][i]);
            }
        }
    } else {
        // The groups' maxima: each lane keeps one group in the first two exchanges (lane / 8), then eight lanes share it.
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
        if ((lane & 7) == 0 && (g0 + lane / 8) * kScaleBlock < d)
            scales[p * s_row + (g0 + lane / 8) * s_group] = mine.s;
        uint8_t* dst = reinterpret_cast<uint8_t*>(q) + p * ldq;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int c = c0 + g * kScaleBlock;
            const float s = __shfl_sync(0xffffffffu, mine.s, 8 * g), r = __shfl_sync(0xffffffffu, mine.r, 8 * g);
            float t[4] = {v[g][0], v[g][1], v[g][2], v[g][3]};
            if (fast) {
                quotient4(t, s, r);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = __fdiv_rn(t[i], s);
            }
            const uint32_t u = to_e4m3x2(t[0], t[1]) | to_e4m3x2(t[2], t[3]) << 16;
            if (VEC) {
                if (c < d) *reinterpret_cast<uint32_t*>(dst + c) = u;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < d) dst[c + i] = (uint8_t)(u >> (8 * i));
            }
        }
    }
}

template <typename SRC, int TYPE>
int launch(const SRC* x, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n, int d, void* q, int64_t ldq,
           float* scales, int64_t s_row, int64_t s_group, unsigned* status, cudaStream_t st)
{
    constexpr int B = TYPE == MB_T_E4M3 ? 1 : 2;
    const bool vec = d % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && (uintptr_t)x % (4 * sizeof(SRC)) == 0 &&
                     (uintptr_t)q % (4 * B) == 0;
    const int cols = kGroups * kScaleBlock;
    const dim3 grid((unsigned)((n + kRowsPerBlock - 1) / kRowsPerBlock), (unsigned)((d + cols - 1) / cols));
    const cudaError_t e =
        vec ? mb_launch_pdl(operand_rows_kernel<SRC, TYPE, true>, grid, dim3(32 * kRowsPerBlock), 0, st, x, ldx, n_src,
                            rows, n, d, q, ldq, scales, s_row, s_group, status)
            : mb_launch_pdl(operand_rows_kernel<SRC, TYPE, false>, grid, dim3(32 * kRowsPerBlock), 0, st, x, ldx, n_src,
                            rows, n, d, q, ldq, scales, s_row, s_group, status);
    if (e != cudaSuccess) return mb_fail(MB_ECUDA, "mb_operand_rows: %s", cudaGetErrorString(e));
    return MB_OK;
}

template <typename SRC>
int launch_as(const SRC* x, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n, int d, int type, void* q,
              int64_t ldq, float* scales, int64_t s_row, int64_t s_group, unsigned* status, cudaStream_t st)
{
    if (type == MB_T_E4M3)
        return launch<SRC, MB_T_E4M3>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status, st);
    if (type == MB_T_BF16)
        return launch<SRC, MB_T_BF16>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status, st);
    return launch<SRC, MB_T_F16>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status, st);
}

}  // namespace

extern "C" int mb_operand_rows(const void* x, int x_type, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n,
                               int d, int type, void* q, int64_t ldq, float* scales, int64_t s_row, int64_t s_group,
                               unsigned* status, void* stream)
{
    MB_REQUIRE(x_type == MB_T_F32 || x_type == MB_T_BF16 || x_type == MB_T_F16, "mb_operand_rows: x type %d", x_type);
    MB_REQUIRE(type == MB_T_E4M3 || type == MB_T_BF16 || type == MB_T_F16, "mb_operand_rows: operand type %d", type);
    MB_REQUIRE(n >= 0 && n < (1ll << 31) && n_src >= 0 && d > 0 && d <= (1 << 24), "mb_operand_rows: n=%lld n_src=%lld d=%d",
               (long long)n, (long long)n_src, d);
    MB_REQUIRE(rows || n <= n_src, "mb_operand_rows: %lld rows of %lld", (long long)n, (long long)n_src);
    MB_REQUIRE(ldx >= d && ldq >= d, "mb_operand_rows: rows closer (%lld, %lld) than their width %d", (long long)ldx,
               (long long)ldq, d);
    if (n == 0) return MB_OK;
    MB_REQUIRE(q && (x || n_src == 0) && (type != MB_T_E4M3 || scales), "mb_operand_rows: null pointer");
    const cudaStream_t st = mb_stream(stream);
    if (x_type == MB_T_F32)
        return launch_as((const float*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status, st);
    if (x_type == MB_T_BF16)
        return launch_as((const __nv_bfloat16*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status,
                      st);
    return launch_as((const __half*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status, st);
}
