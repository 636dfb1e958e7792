// Operand rows: the rows of x picked by index, in the form the float experts'
// products read (e4m3 with one f32 scale per 128 columns, bf16 or f16).
//
// s = max|group| / 448 (448 is e4m3's largest value; 1 for a group of zeros),
// q = e4m3(x / s), both quotients and the cast rounded to nearest even, so the
// largest value of every group maps to +-448 and nothing saturates.
//
// One warp per (row, group): lane l holds columns 4l .. 4l+3.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "mb_common.cuh"
#include "mb_float.cuh"

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }

template <typename SRC, int TYPE>
__global__ void operand_rows_kernel(const SRC* __restrict__ x, int64_t ldx, int64_t n_src,
                                    const int32_t* __restrict__ rows, int64_t n, int d, void* __restrict__ q,
                                    int64_t ldq, float* __restrict__ scales, int64_t s_row, int64_t s_group,
                                    unsigned* status)
{
    const int lane = threadIdx.x & 31;
    const int ng = (d + kScaleBlock - 1) / kScaleBlock;
    const int64_t tasks = n * ng;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); t < tasks; t += step) {
        const int64_t p = t / ng;
        const int g = (int)(t - p * ng);
        const int64_t src = rows ? rows[p] : p;
        const bool ok = src >= 0 && src < n_src;
        if (!ok && lane == 0 && status) atomicOr(status, MB_STATUS_BADARG);
        const int c0 = g * kScaleBlock + 4 * lane;
        float v[4];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = ok && c0 + i < d ? to_f32(x[src * ldx + c0 + i]) : 0.0f;
            m = fmaxf(m, fabsf(v[i]));
        }
        if (TYPE == MB_T_E4M3) {
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = e4m3_scale(m);
            uint8_t* dst = reinterpret_cast<uint8_t*>(q) + p * ldq;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + i < d) dst[c0 + i] = to_e4m3(__fdiv_rn(v[i], s));
            if (lane == 0) scales[p * s_row + g * s_group] = s;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c0 + i < d) store_out<TYPE>(q, p * ldq + c0 + i, v[i]);
        }
    }
}

template <typename SRC>
int launch(const SRC* x, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n, int d, int type, void* q,
           int64_t ldq, float* scales, int64_t s_row, int64_t s_group, unsigned* status, cudaStream_t st)
{
    const int64_t warps = n * ((d + kScaleBlock - 1) / kScaleBlock);
    const unsigned grid = (unsigned)std::min<int64_t>((warps + 7) / 8, (int64_t)mb_num_sms() * 64);
    if (type == MB_T_E4M3)
        operand_rows_kernel<SRC, MB_T_E4M3>
            <<<grid, 256, 0, st>>>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status);
    else if (type == MB_T_BF16)
        operand_rows_kernel<SRC, MB_T_BF16>
            <<<grid, 256, 0, st>>>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status);
    else
        operand_rows_kernel<SRC, MB_T_F16>
            <<<grid, 256, 0, st>>>(x, ldx, n_src, rows, n, d, q, ldq, scales, s_row, s_group, status);
    return mb_check_launch("mb_operand_rows");
}

}  // namespace

extern "C" int mb_operand_rows(const void* x, int x_type, int64_t ldx, int64_t n_src, const int32_t* rows, int64_t n,
                               int d, int type, void* q, int64_t ldq, float* scales, int64_t s_row, int64_t s_group,
                               unsigned* status, void* stream)
{
    MB_REQUIRE(x_type == MB_T_F32 || x_type == MB_T_BF16 || x_type == MB_T_F16, "mb_operand_rows: x type %d", x_type);
    MB_REQUIRE(type == MB_T_E4M3 || type == MB_T_BF16 || type == MB_T_F16, "mb_operand_rows: operand type %d", type);
    MB_REQUIRE(n >= 0 && n < (1ll << 31) && n_src >= 0 && d > 0, "mb_operand_rows: n=%lld n_src=%lld d=%d",
               (long long)n, (long long)n_src, d);
    MB_REQUIRE(rows || n <= n_src, "mb_operand_rows: %lld rows of %lld", (long long)n, (long long)n_src);
    MB_REQUIRE(ldx >= d && ldq >= d, "mb_operand_rows: rows closer (%lld, %lld) than their width %d", (long long)ldx,
               (long long)ldq, d);
    if (n == 0) return MB_OK;
    MB_REQUIRE(q && (x || n_src == 0) && (type != MB_T_E4M3 || scales), "mb_operand_rows: null pointer");
    const cudaStream_t st = mb_stream(stream);
    if (x_type == MB_T_F32)
        return launch((const float*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status, st);
    if (x_type == MB_T_BF16)
        return launch((const __nv_bfloat16*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status,
                      st);
    return launch((const __half*)x, ldx, n_src, rows, n, d, type, q, ldq, scales, s_row, s_group, status, st);
}
