// Root-mean-square norm over the channels of channels-last tensors, with the addition of the residual before it and an output in 8 bits after it.
//
//   s = x + r        y_i = s_i * rsqrt(mean(s^2) + eps) * gain_i        q_i = e4m3(y_i / scale), scale = max(max|y| of the group / 448, 2^-126)
//
// One pass: a token's channels stay in registers between the sum of squares and the product, so that x and r are read once and each output is
// written once.  The bytes bound it (16 x 76 x 76 x 512 bf16, sum and e4m3: 55.7 us, 92 % of the copy rate).  s enters the norm as it was added, in fp32; what is stored of it is rounded once.
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
    int group, group_log2;  // channels that share a scale
    int groups;             // scales of a token
    float eps;
};

constexpr int NORM_VECS = 4;        // 16-byte vectors a thread holds of one token, at most
constexpr int NORM_MAX_WARPS = 32;  // warps of one token

// Two values of a 16-byte vector at a time, as floats.
template <typename T> struct Pairs;
template <> struct Pairs<float> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void get(uint4 v, uint64_t *o)
    {
        o[0] = pack2(__uint_as_float(v.x), __uint_as_float(v.y));
        o[1] = pack2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ uint4 put(const uint64_t *v)
    {
        float x[4];
        unpack2(v[0], x[0], x[1]);
        unpack2(v[1], x[2], x[3]);
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <> struct Pairs<__nv_bfloat16> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(uint4 v, uint64_t *o)
    {
        o[0] = bf16_pair(v.x);
        o[1] = bf16_pair(v.y);
        o[2] = bf16_pair(v.z);
        o[3] = bf16_pair(v.w);
    }
    static __device__ __forceinline__ uint4 put(const uint64_t *v) { return make_uint4(pack_bf16(v[0]), pack_bf16(v[1]), pack_bf16(v[2]), pack_bf16(v[3])); }
};

// The larger of |v|'s two and `most`, as integers: magnitudes of floats are ordered like them, and a NaN is above infinity, so that a token with one says
// so in its scale.
__device__ __forceinline__ uint32_t larger_magnitude(uint64_t v, uint32_t most)
{
    float a, b;
    unpack2(v, a, b);
    return __vimax3_u32(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu, most);
}

// WARPS warps a token (four tokens a block where that is one), VECS 16-byte vectors a thread.  A thread meets the same channels in every token: it keeps
// their gains.  Q: the output in 8 bits.  WHOLE: a token's channels are as many as its threads hold, so that nothing is cut off.
template <typename T, int WARPS, int VECS, bool Q, bool WHOLE>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32, WARPS > 4 ? 1 : VECS <= 2 ? 8 : 5)
rmsnorm_kernel(const __grid_constant__ NormArgs a)
{
    using P = Pairs<T>;
    constexpr int N = 16 / sizeof(T), ROWS = WARPS == 1 ? 4 : 1, LANES = WARPS * 32;
    __shared__ float part[NORM_MAX_WARPS];
    __shared__ uint32_t tops[NORM_MAX_WARPS];
    const int lane = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const int vecs = (a.c + 7) / 8 * 8 / N;
    grid_dependency_wait();
    launch_dependents_if_small();
    const float per_channel = 1.f / (float)a.c;
    uint64_t gain[VECS][P::N];
    const bool wide = a.gain && (uintptr_t)a.gain % 16 == 0;
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (wide && (WHOLE || (lane + k * LANES) * N + N <= a.c)) {
#pragma unroll
            for (int e = 0; e < P::N; e += 2) {
                const float4 g = __ldg(reinterpret_cast<const float4 *>(a.gain + (lane + k * LANES) * N + 2 * e));
                gain[k][e] = pack2(g.x, g.y);
                gain[k][e + 1] = pack2(g.z, g.w);
            }
        } else
#pragma unroll
        for (int e = 0; e < P::N; ++e) {
            const int ch = (lane + k * LANES) * N + 2 * e;
            gain[k][e] = pack2(a.gain && ch < a.c ? __ldg(a.gain + ch) : 1.f, a.gain && ch + 1 < a.c ? __ldg(a.gain + ch + 1) : 1.f);
        }
    // zeros in the place of padding channels, and of what lies behind them
    auto cut = [&](uint64_t *v, int at) {
        if constexpr (!WHOLE) {
            if (at * N + N <= a.c) return;
#pragma unroll
            for (int e = 0; e < P::N; ++e) {
                float lo, hi;
                unpack2(v[e], lo, hi);
                v[e] = pack2(at * N + 2 * e < a.c ? lo : 0.f, at * N + 2 * e + 1 < a.c ? hi : 0.f);
            }
        }
    };
    auto holds = [&](int at) { return WHOLE || at < vecs; };
    long long token = (long long)blockIdx.x * ROWS + (WARPS == 1 ? warp : 0);
    const long long step = (long long)gridDim.x * ROWS;
    const T *px = (const T *)a.x + token * a.xp + lane * N, *pr = (const T *)a.r + token * a.rp + lane * N;
    T *ps = (T *)a.sum + token * a.sp + lane * N, *py = (T *)a.y + token * a.yp + lane * N;
    uint8_t *pq = a.q + token * a.qp + lane * N;
    float *pscale = a.scales + token * a.groups;
    for (; token < a.tokens; token += step, px += step * a.xp, pr += step * a.rp, ps += step * a.sp, py += step * a.yp, pq += step * a.qp, pscale += step * a.groups) {
        uint4 x[VECS], r[VECS];
#pragma unroll
        for (int k = 0; k < VECS; ++k) {                    // all loads of a token in flight together
            x[k] = r[k] = make_uint4(0, 0, 0, 0);
            if (holds(lane + k * LANES)) {
                x[k] = *reinterpret_cast<const uint4 *>(px + k * LANES * N);
                if (a.r) r[k] = *reinterpret_cast<const uint4 *>(pr + k * LANES * N);
            }
        }
        uint64_t v[VECS][P::N], squares2[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < VECS; ++k) {
            const int at = lane + k * LANES;
            uint64_t t[P::N];
            P::get(x[k], v[k]);
            P::get(r[k], t);
#pragma unroll
            for (int e = 0; e < P::N; ++e) v[k][e] = add2(v[k][e], t[e]);       // without a residual: zeros
            cut(v[k], at);
#pragma unroll
            for (int e = 0; e < P::N; ++e) squares2[e & 1] = fma2(v[k][e], v[k][e], squares2[e & 1]);
            if (a.sum && holds(at)) *reinterpret_cast<uint4 *>(ps + k * LANES * N) = P::put(v[k]);
        }
        float squares, odd;
        unpack2(add2(squares2[0], squares2[1]), squares, odd);
        squares += odd;
#pragma unroll
        for (int o = 16; o; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        if (WARPS > 1) {
            if ((threadIdx.x & 31) == 0) part[warp] = squares;
            __syncthreads();
            squares = part[0];
            for (int i = 1; i < WARPS; ++i) squares += part[i];
        }
        const float inv = rsqrtf(fmaf(squares, per_channel, a.eps));
        const uint64_t inv2 = pack2(inv, inv);
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < VECS; ++k) {
            const int at = lane + k * LANES;
#pragma unroll
            for (int e = 0; e < P::N; ++e) v[k][e] = mul2(mul2(v[k][e], inv2), gain[k][e]);
            cut(v[k], at);                                  // ... of a token whose inv is no number
            if (Q && !a.group)
#pragma unroll
                for (int e = 0; e < P::N; ++e) most = larger_magnitude(v[k][e], most);
            if (a.y && holds(at)) *reinterpret_cast<uint4 *>(py + k * LANES * N) = P::put(v[k]);
        }
        if (Q) {
            if (!a.group) {
                most = __reduce_max_sync(0xffffffffu, most);
                if (WARPS > 1) {
                    if ((threadIdx.x & 31) == 0) tops[warp] = most;
                    __syncthreads();
                    most = tops[0];
                    for (int i = 1; i < WARPS; ++i) most = max(most, tops[i]);
                }
            }
#pragma unroll
            for (int k = 0; k < VECS; ++k) {                // every lane of a group is here for the shuffles, whether it holds channels or not
                const int at = lane + k * LANES;
                if (a.group) {
                    most = 0;
#pragma unroll
                    for (int e = 0; e < P::N; ++e) most = larger_magnitude(v[k][e], most);
#pragma unroll
                    for (int o = 1; o < 32; o *= 2)
                        if (o * N < a.group) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                }
                if (!holds(at)) continue;
                // Times the scale's reciprocal, not over the scale: off by an ulp of fp32 or two, where e4m3's half step is 2^-4.
                const float scaled = __uint_as_float(most) * (1.f / 448.f);
                const float scale = scaled < 0x1p-126f ? 0x1p-126f : scaled;    // a NaN stays one
                float to_q;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(to_q) : "f"(scale));
                if (a.group ? (at * N & (a.group - 1)) == 0 : at == 0) pscale[a.group ? at * N >> a.group_log2 : 0] = scale;
                const uint64_t to_q2 = pack2(to_q, to_q);
                uint32_t out[N / 4];
#pragma unroll
                for (int e = 0; e < P::N; e += 2) {
                    float2 lo, hi;
                    unpack2(mul2(v[k][e], to_q2), lo.x, lo.y);
                    unpack2(mul2(v[k][e + 1], to_q2), hi.x, hi.y);
                    out[e / 2] = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
                }
                if (!WHOLE && at * N + N > a.c)             // the padding of a token whose scale is no number is zero all the same
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (at * N + e >= a.c) out[e / 4] &= ~(0xffu << e % 4 * 8);
                uint8_t *to = pq + k * LANES * N;
                if constexpr (N == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1]);
                else *reinterpret_cast<uint32_t *>(to) = out[0];
            }
        }
        if (WARPS > 1) __syncthreads();                     // part[] is read before the next token's
    }
}

template <typename T, int WARPS, int VECS>
static cudaError_t start_rmsnorm(const NormArgs &a, cudaStream_t s)
{
    const long long cap = (long long)sm_count() * (WARPS == 1 ? 8 : 32 / WARPS), blocks = WARPS == 1 ? (a.tokens + 3) / 4 : a.tokens;
    const int grid = (int)(blocks < cap ? blocks : cap), threads = WARPS == 1 ? 128 : WARPS * 32;
    const bool whole = a.c == WARPS * 32 * VECS * (16 / (int)sizeof(T));
    if (a.q) return whole ? launch_overlapped(rmsnorm_kernel<T, WARPS, VECS, true, true>, grid, threads, 0, s, a) : launch_overlapped(rmsnorm_kernel<T, WARPS, VECS, true, false>, grid, threads, 0, s, a);
    return whole ? launch_overlapped(rmsnorm_kernel<T, WARPS, VECS, false, true>, grid, threads, 0, s, a) : launch_overlapped(rmsnorm_kernel<T, WARPS, VECS, false, false>, grid, threads, 0, s, a);
}

// A warp a token while that is enough of it to hold (no barrier), the fewest vectors a thread that hold a token.  No more tokens than SMs: a vector a thread,
// latency is all there is (residual, sum and norm of a token of 1024 channels in bf16: 1.50 us over four warps, 1.83 over one; of 4096 1.83 over 16, 2.25 over 4; over 32 it is slower again).
template <typename T>
static cudaError_t choose_rmsnorm(const NormArgs &a, int vecs, cudaStream_t s)
{
    if (vecs <= 32) return start_rmsnorm<T, 1, 1>(a, s);
    if (a.tokens <= sm_count()) {
        if (vecs <= 128) return start_rmsnorm<T, 4, 1>(a, s);
        if (vecs <= 256) return start_rmsnorm<T, 8, 1>(a, s);
        if (vecs <= 512) return start_rmsnorm<T, 16, 1>(a, s);
    }
    if (vecs <= 64) return start_rmsnorm<T, 1, 2>(a, s);
    if (vecs <= 128) return start_rmsnorm<T, 1, 4>(a, s);
    if (vecs <= 4 * 64) return start_rmsnorm<T, 4, 2>(a, s);
    if (vecs <= 4 * 128) return start_rmsnorm<T, 4, 4>(a, s);
    if (vecs <= 8 * 128) return start_rmsnorm<T, 8, 4>(a, s);
    return start_rmsnorm<T, 32, 4>(a, s);
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
    for (const dnb_tensor *t : {sum, y})
        for (const dnb_tensor *in : {x, residual})
            if (t && in && t->data != in->data && share_memory(t, in)) DNB_FAIL(DNB_EINVAL, "rmsnorm: an output is a part of an input's memory");
    if (sum && y && share_memory(sum, y)) DNB_FAIL(DNB_EINVAL, "rmsnorm: sum and output share memory");
    if (gain && (uintptr_t)gain % 4) DNB_FAIL(DNB_EINVAL, "rmsnorm: gain must be 4-byte aligned");
    for (const dnb_tensor *t : {sum, y})
        if (t && gain && reaches_into(t, gain, (size_t)x->c * 4)) DNB_FAIL(DNB_EINVAL, "rmsnorm: an output is the gain's memory");
    if (!(eps >= 0.f) || eps > 1e30f) DNB_FAIL(DNB_EINVAL, "rmsnorm: eps %g", (double)eps);
    NormArgs a = {};
    if (q) {
        if (!q->data || !q->scales) DNB_FAIL(DNB_EINVAL, "rmsnorm: null e4m3 output");
        if ((uintptr_t)q->data % 16 || (uintptr_t)q->scales % 4) DNB_FAIL(DNB_EINVAL, "rmsnorm: e4m3 data must be 16-byte aligned, its scales 4-byte aligned");
        if (q->pitch < x->c || q->pitch % 8) DNB_FAIL(DNB_EINVAL, "rmsnorm: e4m3 pitch %d for %d channels (need a multiple of 8 >= c)", q->pitch, x->c);
        if (q->group != 0 && q->group != 32 && q->group != 64 && q->group != 128) DNB_FAIL(DNB_EINVAL, "rmsnorm: groups of %d channels (0: one scale a token, 32, 64 or 128)", q->group);
        const size_t tokens = (size_t)x->n * x->h * x->w, values = (tokens - 1) * q->pitch + round_up(x->c, 8), scales = tokens * (q->group ? (x->c + q->group - 1) / q->group : 1) * 4;
        for (const dnb_tensor *t : {x, residual, sum, y})
            if (t && (reaches_into(t, q->data, values) || reaches_into(t, q->scales, scales))) DNB_FAIL(DNB_EINVAL, "rmsnorm: the e4m3 output is another tensor's memory");
        if (ranges_meet(q->data, values, q->scales, scales)) DNB_FAIL(DNB_EINVAL, "rmsnorm: e4m3 values and scales share memory");
        if (gain && (ranges_meet(q->data, values, gain, (size_t)x->c * 4) || ranges_meet(q->scales, scales, gain, (size_t)x->c * 4))) DNB_FAIL(DNB_EINVAL, "rmsnorm: the e4m3 output is the gain's memory");
        a.q = (uint8_t *)q->data; a.scales = q->scales; a.qp = q->pitch; a.group = q->group;
        while (a.group >> a.group_log2 > 1) ++a.group_log2;
        a.groups = q->group ? (x->c + q->group - 1) / q->group : 1;
    }
    const int per_vec = x->dtype == DNB_BF16 ? 8 : 4, vecs = round_up(x->c, 8) / per_vec;
    if (vecs > NORM_MAX_WARPS * 32 * NORM_VECS) DNB_FAIL(DNB_EUNSUPPORTED, "rmsnorm: %d channels (at most %d of this dtype)", x->c, NORM_MAX_WARPS * 32 * NORM_VECS * per_vec);
    a.x = x->data; a.xp = x->cpitch;
    if (residual) { a.r = residual->data; a.rp = residual->cpitch; }
    if (sum) { a.sum = sum->data; a.sp = sum->cpitch; }
    if (y) { a.y = y->data; a.yp = y->cpitch; }
    a.gain = gain; a.eps = eps; a.c = x->c;
    a.tokens = (long long)x->n * x->h * x->w;
    DNB_CUDA(x->dtype == DNB_BF16 ? choose_rmsnorm<__nv_bfloat16>(a, vecs, (cudaStream_t)stream) : choose_rmsnorm<float>(a, vecs, (cudaStream_t)stream));
    DNB_LAUNCH_CHECK("rmsnorm");
    return DNB_OK;
}
