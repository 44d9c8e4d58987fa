// Rotary positions with up to three axes (time, row, column) over channels-last tensors.
//
// A pair (a, b) of a head's channels becomes (a cos t - b sin t, a sin t + b cos t) with t = position * scale * frequency of the axis it belongs to.
// The bytes bound it: every channel is read and written once, and a thread works its sines out once for several heads (16 x 76 x 76 x 1024 bf16: 60.5 us,
// 97 % of the copy rate; one token 4.7 us with a cold cache).
//
// Angles: sine and cosine want t modulo a turn.  A float of t loses that for far positions (position 1e5 has 1/128 of a radian between neighbours),
// so the angle is position * F modulo 2^64, where F is the pair's scale * frequency / 2 pi, its whole turns dropped, in units of 2^-64 turns:
// one integer product, exact modulo a turn.  F itself is off by (1 + |scale * frequency / 2 pi|) * 2^-62 turns at most (its last two bits, and those of a long
// double), the angle by position times that: 2^-30.8 turns for the last position where scale * frequency is 1.
#include <math.h>
#include <string.h>

#include <new>

#include "common.h"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

struct dnb_rope_plan {
    dnb_rope_desc d;
    int pairs;                             // P, over all axes
    uint64_t turn[DNB_ROPE_MAX_PAIRS];     // F of each pair, its last two bits the axis
};

namespace dnb {

constexpr int ROPE_THREADS = 128;

struct RopeArgs {
    uint64_t turn[DNB_ROPE_MAX_PAIRS];
    const void *x;
    void *y;
    const int32_t *positions;              // [tokens][3], or null: the token's place
    unsigned tokens;
    int xp, yp;                            // pitches
    int c, c8;                             // channels, and rounded up to whole vectors of eight
    int h, w, frames, origin[3];
    int heads, head_dim, pairs;
    int chunk, chunks;                     // heads of a thread, and how many such shares a token has
    unsigned turners;                      // blocks that turn; the blocks behind them copy what passes
};

// Sine and cosine of turns * 2^-32 of a turn: the nearest quarter taken off in whole numbers, polynomials of the rest's angle (at most pi / 4) fitted to the
// smallest largest error (4.4e-09 of the sine, 5.1e-10 of the cosine, before rounding).
__device__ __forceinline__ void sine_of(int turns, float &s, float &c)
{
    const int quarter = (int)((unsigned)turns + (1u << 29)) >> 30;
    const float x = (float)(int)((unsigned)turns - ((unsigned)quarter << 30)) * (6.283185307179586f * 0x1p-32f), z = x * x;
    const float sine = fmaf(x * z, fmaf(z, fmaf(z, -0.0001951729936990887f, 0.008332177996635437f), -0.16666655242443085f), x);
    const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.4438451873720624e-05f, -0.001388736767694354f), 0.04166664555668831f), -0.5f), 1.f);
    s = quarter & 1 ? cosine : sine;
    c = quarter & 1 ? sine : cosine;
    if (quarter & 2) s = -s;
    if ((quarter + 1) & 2) c = -c;
}

template <int BYTES> struct RopeVec;
template <> struct RopeVec<2> { using type = uint16_t; };
template <> struct RopeVec<4> { using type = uint32_t; };
template <> struct RopeVec<8> { using type = uint2; };
template <> struct RopeVec<16> { using type = uint4; };

// A thread turns V pairs (V elements at each of two places, a load each) of `chunk` heads of a token; their sines it works out once, in registers.  The
// threads of a warp lie along the pairs of a head, then along shares of heads, then tokens: loads of 16 bytes fill whole sectors.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeArgs a)
{
    using Raw = typename RopeVec<V * (int)sizeof(T)>::type;
    union Vec { Raw raw; T v[V]; };
    constexpr int AT_ONCE = 4;                                                    // heads whose loads are in flight together
    grid_dependency_wait();
    launch_dependents_if_small();
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const int per_head = a.pairs / V;
    if (blockIdx.x < a.turners) {
        const unsigned long long item = (unsigned long long)blockIdx.x * ROPE_THREADS + threadIdx.x;
        const unsigned part = item >> 32 ? (unsigned)(item / (unsigned)per_head) : (unsigned)item / (unsigned)per_head;   // fits: tokens * chunks < 2^31
        const int j = (int)(item - (unsigned long long)part * (unsigned)per_head) * V;
        const unsigned token = part / (unsigned)a.chunks;
        const int head0 = (int)(part - token * (unsigned)a.chunks) * a.chunk;
        if (token >= a.tokens) return;
        const int at_a = INTERLEAVED ? 2 * j : j, apart = INTERLEAVED ? V : a.pairs, count = min(a.chunk, a.heads - head0);
        const T *src = x + (size_t)token * a.xp + head0 * a.head_dim + at_a;
        T *dst = y + (size_t)token * a.yp + head0 * a.head_dim + at_a;
        Vec va[AT_ONCE], vb[AT_ONCE];
        auto load = [&](int h0) {
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h)
                if (h0 + h < count) {
                    va[h].raw = *reinterpret_cast<const Raw *>(src + h * a.head_dim);
                    vb[h].raw = *reinterpret_cast<const Raw *>(src + h * a.head_dim + apart);
                }
        };
        load(0);                                                                  // on their way while the sines are worked out
        long long at[3];
        if (a.positions) {
#pragma unroll
            for (int i = 0; i < 3; ++i) at[i] = a.positions[(size_t)token * 3 + i];
        } else {
            const unsigned row = token / (unsigned)a.w, image = row / (unsigned)a.h;
            at[0] = (long long)(image % (unsigned)a.frames) + a.origin[0];
            at[1] = (long long)(row - image * (unsigned)a.h) + a.origin[1];
            at[2] = (long long)(token - row * (unsigned)a.w) + a.origin[2];
        }
        float cs[V], sn[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint64_t turn = a.turn[j + e];
            const int s = (int)(turn & 3);
            const uint64_t where = (uint64_t)(s == 0 ? at[0] : s == 1 ? at[1] : at[2]);
            const int turns = (int)(where * turn >> 32);                          // signed: from -1/2 to 1/2 of a turn, in units of 2^-32
            // bf16: the hardware's functions, off by 2^-21.41 (sine) and 2^-21.19 (cosine) at most on one turn, where half a step of the output is 2^-9 or more of it
            if (sizeof(T) == 2) __sincosf((float)turns * (6.283185307179586f * 0x1p-32f), &sn[e], &cs[e]);
            else sine_of(turns, sn[e], cs[e]);
        }
        for (int h0 = 0; h0 < count; h0 += AT_ONCE, src += AT_ONCE * a.head_dim, dst += AT_ONCE * a.head_dim) {
            if (h0) load(h0);
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h)
                if (h0 + h < count) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        T &first = INTERLEAVED ? (2 * e < V ? va[h].v[(2 * e) % V] : vb[h].v[(2 * e) % V]) : va[h].v[e];
                        T &second = INTERLEAVED ? (2 * e + 1 < V ? va[h].v[(2 * e + 1) % V] : vb[h].v[(2 * e + 1) % V]) : vb[h].v[e];
                        const float p = to_float<T>(first), q = to_float<T>(second);
                        first = from_float<T>(p * cs[e] - q * sn[e]);
                        second = from_float<T>(p * sn[e] + q * cs[e]);
                    }
                    *reinterpret_cast<Raw *>(dst + h * a.head_dim) = va[h].raw;
                    *reinterpret_cast<Raw *>(dst + h * a.head_dim + apart) = vb[h].raw;
                }
        }
        return;
    }
    // What passes: of each head the channels behind its pairs, by V, and the channels behind the heads, by eights (by one where they start off a vector).
    const int rest = (a.head_dim - 2 * a.pairs) / V, tail0 = a.heads * a.head_dim, unit = tail0 & 7 ? 1 : 8, tail = (a.c8 - tail0) / unit;
    const unsigned per_token = (unsigned)(a.heads * rest + tail);
    const unsigned long long total = (unsigned long long)a.tokens * per_token, step = (unsigned long long)(gridDim.x - a.turners) * ROPE_THREADS;
    for (unsigned long long i = (unsigned long long)(blockIdx.x - a.turners) * ROPE_THREADS + threadIdx.x; i < total; i += step) {
        const unsigned token = (unsigned)(i / per_token);
        const int r = (int)(i - (unsigned long long)token * per_token);
        const T *src = x + (size_t)token * a.xp;
        T *dst = y + (size_t)token * a.yp;
        if (r < a.heads * rest) {
            const int at = r / rest * a.head_dim + 2 * a.pairs + r % rest * V;
            *reinterpret_cast<Raw *>(dst + at) = *reinterpret_cast<const Raw *>(src + at);
        } else if (unit == 1) {
            const int at = tail0 + r - a.heads * rest;
            dst[at] = at < a.c ? src[at] : from_float<T>(0.f);
        } else {
            const int at = tail0 + (r - a.heads * rest) * 8;
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int b = 0; b < 8 / N; ++b) {                                     // eight channels: one vector of bf16, two of f32
                union { uint4 raw; T v[N]; } v;
                v.raw = reinterpret_cast<const uint4 *>(src + at)[b];
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (at + b * N + e >= a.c) v.v[e] = from_float<T>(0.f);       // padding channels stay zero
                reinterpret_cast<uint4 *>(dst + at)[b] = v.raw;
            }
        }
    }
}

template <typename T, int V>
static cudaError_t start_rope(const RopeArgs &a, bool interleaved, unsigned grid, cudaStream_t s)
{
    return interleaved ? launch_overlapped(rope_kernel<T, V, true>, grid, ROPE_THREADS, 0, s, a) : launch_overlapped(rope_kernel<T, V, false>, grid, ROPE_THREADS, 0, s, a);
}

static int launch_rope(const dnb_rope_plan &p, const dnb_tensor *x, const int32_t *positions, const dnb_tensor *y, cudaStream_t s)
{
    const dnb_rope_desc &d = p.d;
    DNB_TRY(check_tensor(x, "rope input"));
    DNB_TRY(check_tensor(y, "rope output"));
    if (x->layout != DNB_NHWC || y->layout != DNB_NHWC) DNB_FAIL(DNB_EINVAL, "rope: tensors must be channels-last");
    if (x->dtype != y->dtype || x->n != y->n || x->h != y->h || x->w != y->w || x->c != y->c) DNB_FAIL(DNB_EINVAL, "rope: input and output differ in dtype or extents");
    if ((long long)d.heads * d.head_dim > x->c) DNB_FAIL(DNB_EINVAL, "rope: %d heads of %d channels in a tensor of %d", d.heads, d.head_dim, x->c);
    if (x->data == y->data && x->cpitch != y->cpitch) DNB_FAIL(DNB_EINVAL, "rope: in place with another cpitch");
    if (x->data != y->data && share_memory(x, y)) DNB_FAIL(DNB_EINVAL, "rope: the output is a part of the input's memory");
    if (positions && (uintptr_t)positions % 4) DNB_FAIL(DNB_EINVAL, "rope: positions must be 4-byte aligned");
    if (!positions && x->n % d.frames) DNB_FAIL(DNB_EINVAL, "rope: %d images are no whole number of clips of %d frames", x->n, d.frames);
    const long long tokens = (long long)x->n * x->h * x->w;
    if ((long long)x->n * x->h >= 1LL << 31 || tokens >= 1LL << 31) DNB_FAIL(DNB_EUNSUPPORTED, "rope: 2^31 tokens or more");
    if (positions && reaches_into(y, positions, (size_t)tokens * 12)) DNB_FAIL(DNB_EINVAL, "rope: the output is the positions' memory");
    RopeArgs a;
    memcpy(a.turn, p.turn, sizeof(a.turn));
    a.x = x->data; a.y = y->data; a.positions = positions;
    a.tokens = (unsigned)tokens;
    a.xp = x->cpitch; a.yp = y->cpitch;
    a.c = x->c; a.c8 = round_up(x->c, 8);
    a.h = x->h; a.w = x->w; a.frames = d.frames;
    for (int i = 0; i < 3; ++i) a.origin[i] = d.origin[i];
    a.heads = d.heads; a.head_dim = d.head_dim; a.pairs = p.pairs;
    // the widest vector that the pairs and the heads are whole numbers of
    int v = x->dtype == DNB_BF16 ? 8 : 4;
    while (p.pairs % v || d.head_dim % v) v /= 2;
    // Heads of a thread: eight, so that its sines cost it little; fewer while the GPU has room for the threads, two blocks an SM (a grid of that size starts
    // early, see launch_overlapped).
    const int per_head = p.pairs / v;
    auto threads = [&](int chunk) { return tokens * per_head * ((d.heads + chunk - 1) / chunk); };
    a.chunk = d.heads < 8 ? d.heads : 8;
    while (a.chunk > 1 && threads((a.chunk + 1) / 2) <= (long long)sm_count() * 2 * ROPE_THREADS) a.chunk = (a.chunk + 1) / 2;
    a.chunks = (d.heads + a.chunk - 1) / a.chunk;
    if (tokens * a.chunks >= 1LL << 31) { a.chunk = d.heads; a.chunks = 1; }
    const unsigned long long turners = ((unsigned long long)tokens * a.chunks * per_head + ROPE_THREADS - 1) / ROPE_THREADS;
    const long long passing = x->data == y->data ? 0 : d.heads * (long long)((d.head_dim - 2 * p.pairs) / v) + (a.c8 - d.heads * d.head_dim + 7) / 8;
    const long long copiers = (tokens * passing + 4 * ROPE_THREADS - 1) / (4 * ROPE_THREADS), most = (long long)sm_count() * 16;
    if (turners + most >= 1ULL << 31) DNB_FAIL(DNB_EUNSUPPORTED, "rope: %lld tokens", tokens);
    a.turners = (unsigned)turners;
    const unsigned grid = a.turners + (unsigned)(copiers < most ? copiers : most);
    cudaError_t e;
    if (x->dtype == DNB_BF16) {
        using T = __nv_bfloat16;
        e = v == 8 ? start_rope<T, 8>(a, d.interleaved, grid, s) : v == 4 ? start_rope<T, 4>(a, d.interleaved, grid, s)
            : v == 2 ? start_rope<T, 2>(a, d.interleaved, grid, s) : start_rope<T, 1>(a, d.interleaved, grid, s);
    } else {
        e = v == 4 ? start_rope<float, 4>(a, d.interleaved, grid, s) : v == 2 ? start_rope<float, 2>(a, d.interleaved, grid, s) : start_rope<float, 1>(a, d.interleaved, grid, s);
    }
    DNB_CUDA(e);
    DNB_LAUNCH_CHECK("rope");
    return DNB_OK;
}

}  // namespace dnb

using namespace dnb;

extern "C" int dnb_rope_plan_create(const dnb_rope_desc *desc, dnb_rope_plan **plan)
{
    if (!desc || !plan) DNB_FAIL(DNB_EINVAL, "rope: null argument");
    *plan = nullptr;
    const dnb_rope_desc &d = *desc;
    long long pairs = 0;
    for (int i = 0; i < 3; ++i) {
        if (d.pairs[i] < 0) DNB_FAIL(DNB_EINVAL, "rope: %d pairs for axis %d", d.pairs[i], i);
        if (!isfinite(d.scale[i])) DNB_FAIL(DNB_EINVAL, "rope: scale of axis %d is not finite", i);
        pairs += d.pairs[i];
    }
    if (d.head_dim < 2 || d.head_dim % 2 || d.heads < 1) DNB_FAIL(DNB_EINVAL, "rope: %d heads of %d channels", d.heads, d.head_dim);
    if (pairs < 1 || 2 * pairs > d.head_dim) DNB_FAIL(DNB_EINVAL, "rope: %lld pairs in a head of %d channels", pairs, d.head_dim);
    if (pairs > DNB_ROPE_MAX_PAIRS) DNB_FAIL(DNB_EUNSUPPORTED, "rope: %lld pairs (at most %d)", pairs, DNB_ROPE_MAX_PAIRS);
    if (!(d.base > 0.f) || !isfinite(d.base)) DNB_FAIL(DNB_EINVAL, "rope: base %g", (double)d.base);
    if (d.frames < 1) DNB_FAIL(DNB_EINVAL, "rope: %d frames", d.frames);
    if ((d.interleaved | d.shared) & ~1) DNB_FAIL(DNB_EINVAL, "rope: interleaved %d, shared %d (0 or 1)", d.interleaved, d.shared);
    dnb_rope_plan *p = new (std::nothrow) dnb_rope_plan();
    if (!p) DNB_FAIL(DNB_ENOMEM, "rope: no memory for the plan");
    p->d = d;
    p->pairs = (int)pairs;
    int i = 0;
    for (int axis = 0; axis < 3; ++axis)
        for (int j = 0; j < d.pairs[axis]; ++j, ++i) {
            const long double power = d.shared ? (long double)i / pairs : (long double)j / d.pairs[axis];
            const long double per_step = powl((long double)d.base, -power) * d.scale[axis] / (2 * 3.141592653589793238462643383279502884L);
            const long double turn = per_step - floorl(per_step);                 // 0 <= turn < 1 (1 if it rounds up)
            p->turn[i] = ((turn * 0x1p64L >= 0x1p64L ? 0 : (uint64_t)(turn * 0x1p64L)) & ~3ULL) | (uint64_t)axis;
        }
    *plan = p;
    return DNB_OK;
}

extern "C" void dnb_rope_plan_destroy(dnb_rope_plan *plan) { delete plan; }

extern "C" int dnb_rope_forward(const dnb_rope_plan *plan, const dnb_tensor *x, const int32_t *positions, const dnb_tensor *y, void *stream)
{
    if (!plan) DNB_FAIL(DNB_EINVAL, "rope: null plan");
    return launch_rope(*plan, x, positions, y, (cudaStream_t)stream);
}
