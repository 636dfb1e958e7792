// Products of rows grouped by expert with each expert's float matrix (e4m3 with
// block scales, bf16 or f16), and the gate|up form with SiLU(gate) * up.
//
//   y[p, o] = sum_g xs[p, g] ws[e, o / 128, g] sum_{k in g} x[p, k] w[e, o, k]
//
// with g over groups of 128 columns (one group, scales 1, for 16-bit types).
// Products of e4m3 values are exact in f32; each group's sum is scaled in f32.
//
// One CTA per (row, 128 outputs): the row's group of 128 columns in shared
// memory, one output per thread.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "mb_common.cuh"
#include "mb_float.cuh"

namespace {

struct GroupedArgs {
    const void* x;
    int64_t ldx;
    const float* xs;
    int64_t xs_row, xs_group;
    int64_t P;
    const void* w;
    int64_t w_expert, ldw;
    const float* ws;
    int E, O, K;               // O: output rows of w (I for the gate|up form, whose matrices have 2I)
    const int32_t* offsets;    // null: one expert, all rows
    void* y;
    int64_t ldy;
    float* qs;
    int64_t qs_row, qs_group;
    unsigned* status;
};

template <int TYPE>
__device__ __forceinline__ float load_elem(const void* p, int64_t i)
{
    if (TYPE == MB_T_E4M3) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(reinterpret_cast<const uint8_t*>(p)[i], __NV_E4M3);
        return __half2float(__half(h));
    }
    if (TYPE == MB_T_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

// The rows of expert e, or none where the offsets are not what they may be (reported).
__device__ __forceinline__ int2 expert_rows(const GroupedArgs& a, int e)
{
    if (!a.offsets) return make_int2(0, (int)a.P);
    const int lo = a.offsets[e], hi = a.offsets[e + 1];
    if (lo < 0 || hi < lo || hi > a.P) {
        if (a.status) atomicOr(a.status, MB_STATUS_BADARG);
        return make_int2(0, 0);
    }
    return make_int2(lo, hi);
}

template <int TYPE, int OUT, bool SWIGLU>
__global__ void grouped_kernel(const GroupedArgs a)
{
    __shared__ float xrow[kScaleBlock];
    __shared__ float red[4];
    const int o = blockIdx.x * 128 + threadIdx.x;
    const int Kb = (a.K + kScaleBlock - 1) / kScaleBlock, Ob = (a.O + kScaleBlock - 1) / kScaleBlock;
    for (int64_t p = blockIdx.y; p < a.P; p += gridDim.y) {
        int e = -1;
        for (int i = 0; i < a.E; ++i) {
            const int2 r = expert_rows(a, i);
            if (p >= r.x && p < r.y) {
                e = i;
                break;
            }
        }
        if (e < 0) continue;
        float acc[2] = {0.0f, 0.0f};
        for (int kb = 0; kb < Kb; ++kb) {
            const int k0 = kb * kScaleBlock, kn = min(kScaleBlock, a.K - k0);
            __syncthreads();
            xrow[threadIdx.x] = (int)threadIdx.x < kn ? load_elem<TYPE>(a.x, p * a.ldx + k0 + threadIdx.x) : 0.0f;
            __syncthreads();
            if (o >= a.O) continue;
#pragma unroll
            for (int h = 0; h < (SWIGLU ? 2 : 1); ++h) {
                const int64_t row = (int64_t)e * a.w_expert + (int64_t)(h * a.O + o) * a.ldw + k0;
                float sum = 0.0f;
                for (int k = 0; k < kn; ++k) sum = fmaf(xrow[k], load_elem<TYPE>(a.w, row + k), sum);
                if (TYPE == MB_T_E4M3)
                    sum *= a.xs[p * a.xs_row + kb * a.xs_group] *
                           a.ws[(((int64_t)e * (SWIGLU ? 2 : 1) + h) * Ob + o / kScaleBlock) * Kb + kb];
                acc[h] += sum;
            }
        }
        if (!SWIGLU) {
            if (o < a.O) store_out<OUT>(a.y, p * a.ldy + o, acc[0]);
            continue;
        }
        const float act = o < a.O ? acc[0] / (1.0f + expf(-acc[0])) * acc[1] : 0.0f;
        if (TYPE != MB_T_E4M3) {
            if (o < a.O) store_out<OUT>(a.y, p * a.ldy + o, act);
            continue;
        }
        float m = fabsf(act);
        for (int s = 16; s; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        const float s = e4m3_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        if (o < a.O) reinterpret_cast<uint8_t*>(a.y)[p * a.ldy + o] = to_e4m3(__fdiv_rn(act, s));
        if (threadIdx.x == 0) a.qs[p * a.qs_row + blockIdx.x * a.qs_group] = s;
    }
}

template <int TYPE, int OUT, bool SWIGLU>
int launch(const GroupedArgs& a, const char* what, cudaStream_t st)
{
    const dim3 grid((a.O + 127) / 128, (unsigned)std::min<int64_t>(a.P, 65535));
    grouped_kernel<TYPE, OUT, SWIGLU><<<grid, 128, 0, st>>>(a);
    return mb_check_launch(what);
}

template <int TYPE>
int run_matmul(const GroupedArgs& a, int y_type, const char* what, cudaStream_t st)
{
    if (y_type == MB_T_F32) return launch<TYPE, MB_T_F32, false>(a, what, st);
    if (y_type == MB_T_BF16) return launch<TYPE, MB_T_BF16, false>(a, what, st);
    return launch<TYPE, MB_T_F16, false>(a, what, st);
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

int matmul(const GroupedArgs& a, int type, int y_type, const char* what, void* stream)
{
    MB_REQUIRE(y_type == MB_T_F32 || y_type == MB_T_BF16 || y_type == MB_T_F16, "%s: result type %d", what, y_type);
    int rc = check_args(a, type, 1, what);
    if (rc || a.P == 0) return rc;
    const cudaStream_t st = mb_stream(stream);
    if (type == MB_T_E4M3) return run_matmul<MB_T_E4M3>(a, y_type, what, st);
    if (type == MB_T_BF16) return run_matmul<MB_T_BF16>(a, y_type, what, st);
    return run_matmul<MB_T_F16>(a, y_type, what, st);
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
    if (type == MB_T_E4M3) return launch<MB_T_E4M3, MB_T_F32, true>(a, what, st);
    if (type == MB_T_BF16) return launch<MB_T_BF16, MB_T_BF16, true>(a, what, st);
    return launch<MB_T_F16, MB_T_F16, true>(a, what, st);
}
