// Root-mean-square norm over the channels of channels-last tensors, with the addition of the residual before it and an output in 8 bits after it.
//
//   s = x + r        y_i = s_i * rsqrt(mean(s^2) + eps) * gain_i        q_i = e4m3(y_i / scale), scale = max(max|y| of the group / 448, 2^-126)
//
// One pass: a token's channels stay in registers between the sum of squares and the product, so that x and r are read once and each output is
// written once.  The bytes bound it.  s enters the norm as it was added, in fp32; what is stored of it is rounded once.
#include <cuda_fp8.h>

#include "common.h"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

namespace dnb {

struct NormArgs {
    const void *x, *r;      // r may be null
    const float *gain;      // [c], or null: 1
    void *sum, *y;          // either may be null
    uint8_t *q;             // may be null
    float *scales;
    long long tokens;
    int c, xp, rp, sp, yp, qp;
    int group, groups;      // channels that share a scale, and how many scales a token has
    float eps;
};

constexpr int NORM_VECS = 4;        // 16-byte vectors a thread holds of one token
constexpr int NORM_MAX_WARPS = 32;  // warps of one token

// max that a NaN wins, so that a token with one says so in its scale
__device__ __forceinline__ float max_nan(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// WARPS warps a token, several tokens a block where that is one.
template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32)
rmsnorm_kernel(const __grid_constant__ NormArgs a)
{
    constexpr int N = 16 / sizeof(T), ROWS = WARPS == 1 ? 4 : 1, LANES = WARPS * 32;
    union Vec { uint4 raw; T v[N]; };
    __shared__ float part[2][NORM_MAX_WARPS];
    grid_dependency_wait();
    launch_dependents_if_small();
    const int lane = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const int vecs = (a.c + 7) / 8 * 8 / N;
    for (long long token = (long long)blockIdx.x * ROWS + (WARPS == 1 ? warp : 0); token < a.tokens; token += (long long)gridDim.x * ROWS) {
        float v[NORM_VECS][N];
        float squares = 0.f;
#pragma unroll
        for (int k = 0; k < NORM_VECS; ++k) {
            const int at = lane + k * LANES;
            if (at >= vecs) break;
            Vec x, r;
            x.raw = reinterpret_cast<const uint4 *>((const T *)a.x + (size_t)token * a.xp)[at];
            if (a.r) r.raw = reinterpret_cast<const uint4 *>((const T *)a.r + (size_t)token * a.rp)[at];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                v[k][e] = to_float<T>(x.v[e]);
                if (a.r) v[k][e] += to_float<T>(r.v[e]);
                if (at * N + e >= a.c) v[k][e] = 0.f;       // padding channels
            }
            if (a.sum) {
                Vec o;
#pragma unroll
                for (int e = 0; e < N; ++e) o.v[e] = from_float<T>(v[k][e]);
                reinterpret_cast<uint4 *>((T *)a.sum + (size_t)token * a.sp)[at] = o.raw;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) squares = fmaf(v[k][e], v[k][e], squares);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        if (WARPS > 1) {
            if ((threadIdx.x & 31) == 0) part[0][warp] = squares;
            __syncthreads();
            squares = part[0][0];
            for (int i = 1; i < WARPS; ++i) squares += part[0][i];
        }
        const float inv = 1.f / sqrtf(squares / (float)a.c + a.eps);
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < NORM_VECS; ++k) {
            const int at = lane + k * LANES;
            if (at >= vecs) break;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int ch = at * N + e;
                v[k][e] *= inv;
                if (a.gain && ch < a.c) v[k][e] *= __ldg(a.gain + ch);
                if (ch >= a.c) v[k][e] = 0.f;               // ... of a token whose inv is no number
                most = max_nan(most, fabsf(v[k][e]));
            }
            if (a.y) {
                Vec o;
#pragma unroll
                for (int e = 0; e < N; ++e) o.v[e] = from_float<T>(v[k][e]);
                reinterpret_cast<uint4 *>((T *)a.y + (size_t)token * a.yp)[at] = o.raw;
            }
        }
        if (a.q) {
            if (!a.group) {
#pragma unroll
                for (int o = 16; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (WARPS > 1) {
                    if ((threadIdx.x & 31) == 0) part[1][warp] = most;
                    __syncthreads();
                    most = part[1][0];
                    for (int i = 1; i < WARPS; ++i) most = max_nan(most, part[1][i]);
                }
            }
#pragma unroll
            for (int k = 0; k < NORM_VECS; ++k) {
                const int at = lane + k * LANES;
                if (k * LANES >= vecs) break;               // by whole rounds: the lanes of a group meet in the shuffles
                if (a.group) {
                    most = 0.f;
                    if (at < vecs)
#pragma unroll
                        for (int e = 0; e < N; ++e) most = max_nan(most, fabsf(v[k][e]));
                    for (int o = a.group / N / 2; o; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
                }
                if (at >= vecs) continue;
                const float scale = max_nan(most / 448.f, 0x1p-126f);
                const int g = a.group ? at * N / a.group : 0;
                if (a.group ? at * N % a.group == 0 : at == 0) a.scales[(size_t)token * a.groups + g] = scale;
                uint32_t out[N / 4];
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[k][e] / scale, v[k][e + 1] / scale), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[k][e + 2] / scale, v[k][e + 3] / scale), __NV_SATFINITE, __NV_E4M3);
                    out[e / 4] = lo | hi << 16;
                }
#pragma unroll
                for (int e = 0; e < N; ++e)                 // the padding of a token whose scale is no number is zero all the same
                    if (at * N + e >= a.c) out[e / 4] &= ~(0xffu << e % 4 * 8);
                uint8_t *to = a.q + (size_t)token * a.qp + at * N;
                if constexpr (N == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1]);
                else *reinterpret_cast<uint32_t *>(to) = out[0];
            }
        }
        if (WARPS > 1) __syncthreads();                     // part[] is read before the next token's
    }
}

template <typename T>
static cudaError_t start_rmsnorm(const NormArgs &a, int warps, cudaStream_t s)
{
    const long long cap = (long long)sm_count() * (warps == 1 ? 16 : 64 / warps), blocks = warps == 1 ? (a.tokens + 3) / 4 : a.tokens;
    const int grid = (int)(blocks < cap ? blocks : cap);
    switch (warps) {
    case 1: return launch_overlapped(rmsnorm_kernel<T, 1>, grid, 128, 0, s, a);
    case 4: return launch_overlapped(rmsnorm_kernel<T, 4>, grid, 128, 0, s, a);
    case 8: return launch_overlapped(rmsnorm_kernel<T, 8>, grid, 256, 0, s, a);
    default: return launch_overlapped(rmsnorm_kernel<T, 32>, grid, 1024, 0, s, a);
    }
}

// A tensor of the norm: channels-last with x's extents and dtype; one that is x's own memory has its pitch too.
static int check_norm_tensor(const dnb_tensor *x, const dnb_tensor *t, const char *what)
{
    DNB_TRY(check_tensor(t, what));
    if (t->layout != DNB_NHWC || t->dtype != x->dtype) DNB_FAIL(DNB_EINVAL, "%s: must be channels-last with the input's dtype", what);
    if (t->n != x->n || t->h != x->h || t->w != x->w || t->c != x->c) DNB_FAIL(DNB_EINVAL, "%s: extents differ from the input's", what);
    if (t->data == x->data && t->cpitch != x->cpitch) DNB_FAIL(DNB_EINVAL, "%s: in place with another cpitch", what);
    return DNB_OK;
}

}  // namespace dnb

using namespace dnb;

extern "C" int dnb_rmsnorm_forward(const dnb_tensor *x, const dnb_tensor *residual, const float *gain, float eps, const dnb_tensor *sum,
                                   const dnb_tensor *y, const dnb_e4m3 *q, void *stream)
{
    DNB_TRY(check_tensor(x, "rmsnorm input"));
    if (x->layout != DNB_NHWC) DNB_FAIL(DNB_EINVAL, "rmsnorm: tensors must be channels-last");
    if (!sum && !y && !q) DNB_FAIL(DNB_EINVAL, "rmsnorm: no output");
    if (residual) DNB_TRY(check_norm_tensor(x, residual, "rmsnorm residual"));
    if (sum) DNB_TRY(check_norm_tensor(x, sum, "rmsnorm sum"));
    if (y) DNB_TRY(check_norm_tensor(x, y, "rmsnorm output"));
    if (sum && !residual) DNB_FAIL(DNB_EINVAL, "rmsnorm: a sum without a residual");
    if (sum && y && sum->data == y->data) DNB_FAIL(DNB_EINVAL, "rmsnorm: sum and output are one tensor");
    for (const dnb_tensor *t : {sum, y})
        if (t && residual && t->data == residual->data && t->cpitch != residual->cpitch) DNB_FAIL(DNB_EINVAL, "rmsnorm: in place with another cpitch");
    if (gain && (uintptr_t)gain % 4) DNB_FAIL(DNB_EINVAL, "rmsnorm: gain must be 4-byte aligned");
    if (!(eps >= 0.f) || eps > 1e30f) DNB_FAIL(DNB_EINVAL, "rmsnorm: eps %g", (double)eps);
    NormArgs a = {};
    if (q) {
        if (!q->data || !q->scales) DNB_FAIL(DNB_EINVAL, "rmsnorm: null e4m3 output");
        if ((uintptr_t)q->data % 16 || (uintptr_t)q->scales % 4) DNB_FAIL(DNB_EINVAL, "rmsnorm: e4m3 data must be 16-byte aligned, its scales 4-byte aligned");
        if (q->pitch < x->c || q->pitch % 8) DNB_FAIL(DNB_EINVAL, "rmsnorm: e4m3 pitch %d for %d channels (need a multiple of 8 >= c)", q->pitch, x->c);
        if (q->group != 0 && q->group != 32 && q->group != 64 && q->group != 128) DNB_FAIL(DNB_EINVAL, "rmsnorm: groups of %d channels (0: one scale a token, 32, 64 or 128)", q->group);
        for (const dnb_tensor *t : {x, residual, sum, y})
            if (t && (t->data == q->data || t->data == (void *)q->scales)) DNB_FAIL(DNB_EINVAL, "rmsnorm: the e4m3 output is another tensor's memory");
        a.q = (uint8_t *)q->data; a.scales = q->scales; a.qp = q->pitch; a.group = q->group;
        a.groups = q->group ? (x->c + q->group - 1) / q->group : 1;
    }
    const int per_vec = x->dtype == DNB_BF16 ? 8 : 4, vecs = round_up(x->c, 8) / per_vec, need = (vecs + 32 * NORM_VECS - 1) / (32 * NORM_VECS);
    if (need > NORM_MAX_WARPS) DNB_FAIL(DNB_EUNSUPPORTED, "rmsnorm: %d channels (at most %d of this dtype)", x->c, NORM_MAX_WARPS * 32 * NORM_VECS * per_vec);
    a.x = x->data; a.xp = x->cpitch;
    if (residual) { a.r = residual->data; a.rp = residual->cpitch; }
    if (sum) { a.sum = sum->data; a.sp = sum->cpitch; }
    if (y) { a.y = y->data; a.yp = y->cpitch; }
    a.gain = gain; a.eps = eps; a.c = x->c;
    a.tokens = (long long)x->n * x->h * x->w;
    const int warps = need == 1 ? 1 : need <= 4 ? 4 : need <= 8 ? 8 : 32;
    DNB_CUDA(x->dtype == DNB_BF16 ? start_rmsnorm<__nv_bfloat16>(a, warps, (cudaStream_t)stream) : start_rmsnorm<float>(a, warps, (cudaStream_t)stream));
    DNB_LAUNCH_CHECK("rmsnorm");
    return DNB_OK;
}
