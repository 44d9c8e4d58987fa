// Rotary positions with up to three axes (time, row, column) over channels-last tensors.
//
// A pair (a, b) of a head's channels becomes (a cos t - b sin t, a sin t + b cos t) with t = position * scale * frequency of the axis it belongs to.
// The bytes bound it: every channel is read and written once, and a token's sines are computed once for all of its heads (a table in shared
// memory), not once per element.
//
// Angles: sine and cosine want t modulo a turn.  A float of t loses that for far positions (position 1e5 has 1/128 of a radian between neighbours),
// so the table entry is position * F modulo 2^64, where F is the pair's scale * frequency / 2 pi, its whole turns dropped, in units of 2^-64 turns:
// one integer product, exact modulo a turn, off by at most position * 2^-65 turns however far the position is.
#include <math.h>
#include <string.h>

#include <new>

#include "common.h"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

struct dnb_rope_plan {
    dnb_rope_desc d;
    int pairs;                             // P, over all axes
    uint64_t turn[DNB_ROPE_MAX_PAIRS];     // F of each pair
    uint8_t axis[DNB_ROPE_MAX_PAIRS];
};

namespace dnb {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_TABLE = 2048;           // sines and cosines that a block holds: 16 KB

struct RopeArgs {
    uint64_t turn[DNB_ROPE_MAX_PAIRS];
    uint8_t axis[DNB_ROPE_MAX_PAIRS];
    const void *x;
    void *y;
    const int32_t *positions;              // [tokens][3], or null: the token's place
    long long tokens;
    int xp, yp;                            // pitches
    int c, c8;                             // channels, and rounded up to whole vectors of eight
    int h, w, frames, origin[3];
    int heads, head_dim, pairs;
    int tile;                              // tokens whose table a block holds at a time
};

template <int BYTES> struct RopeVec;
template <> struct RopeVec<2> { using type = uint16_t; };
template <> struct RopeVec<4> { using type = uint32_t; };
template <> struct RopeVec<8> { using type = uint2; };
template <> struct RopeVec<16> { using type = uint4; };

// V pairs an item: V elements at each of two places, in one load each.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeArgs a)
{
    using Raw = typename RopeVec<V * (int)sizeof(T)>::type;
    union Vec { Raw raw; T v[V]; };
    __shared__ float2 table[ROPE_TABLE];
    grid_dependency_wait();
    launch_dependents_if_small();
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const bool copies = a.x != a.y;
    const int per_head = a.pairs / V, per_token = a.heads * per_head;
    const int rest = (a.head_dim - 2 * a.pairs) / V;                              // vectors of a head that do not turn
    const int tail0 = a.heads * a.head_dim, tail = (a.c8 - tail0) / 8;            // channels behind the heads, by eights
    const long long tiles = (a.tokens + a.tile - 1) / a.tile;
    for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const long long first = t * a.tile;
        const int count = (int)(a.tokens - first < a.tile ? a.tokens - first : a.tile);
        __syncthreads();                                                          // the last tile's table has been read
        for (int i = threadIdx.x; i < count * a.pairs; i += ROPE_THREADS) {
            const int k = i / a.pairs, pair = i - k * a.pairs, axis = a.axis[pair];
            const long long token = first + k;
            long long at;
            if (a.positions) at = a.positions[token * 3 + axis];
            else {
                const int row = (int)(token / a.w);
                at = axis == 2 ? token - (long long)row * a.w : axis == 1 ? row % a.h : row / a.h % a.frames;
                at += a.origin[axis];
            }
            const int turns = (int)((uint64_t)at * a.turn[pair] >> 32);           // signed: from -1/2 to 1/2 of a turn, in units of 2^-32
            float s, c;
            sincospif((float)turns * 0x1p-31f, &s, &c);
            table[i] = make_float2(c, s);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count * per_token; i += ROPE_THREADS) {
            const int k = i / per_token, r = i - k * per_token;
            const int head = r / per_head, j = (r - head * per_head) * V;
            const int at_a = head * a.head_dim + (INTERLEAVED ? 2 * j : j), at_b = at_a + (INTERLEAVED ? V : a.pairs);
            const T *src = x + (size_t)(first + k) * a.xp;
            T *dst = y + (size_t)(first + k) * a.yp;
            Vec va, vb;
            va.raw = *reinterpret_cast<const Raw *>(src + at_a);
            vb.raw = *reinterpret_cast<const Raw *>(src + at_b);
            const float2 *cs = table + k * a.pairs + j;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                T &first_of = INTERLEAVED ? (2 * e < V ? va.v[(2 * e) % V] : vb.v[(2 * e) % V]) : va.v[e];
                T &second_of = INTERLEAVED ? (2 * e + 1 < V ? va.v[(2 * e + 1) % V] : vb.v[(2 * e + 1) % V]) : vb.v[e];
                const float p = to_float<T>(first_of), q = to_float<T>(second_of);
                first_of = from_float<T>(p * cs[e].x - q * cs[e].y);
                second_of = from_float<T>(p * cs[e].y + q * cs[e].x);
            }
            *reinterpret_cast<Raw *>(dst + at_a) = va.raw;
            *reinterpret_cast<Raw *>(dst + at_b) = vb.raw;
        }
        if (!copies) continue;
        for (int i = threadIdx.x; i < count * a.heads * rest; i += ROPE_THREADS) {
            const int k = i / (a.heads * rest), r = i - k * a.heads * rest;
            const int at = r / rest * a.head_dim + 2 * a.pairs + r % rest * V;
            *reinterpret_cast<Raw *>(y + (size_t)(first + k) * a.yp + at) = *reinterpret_cast<const Raw *>(x + (size_t)(first + k) * a.xp + at);
        }
        if ((tail0 & 7) == 0) {
            for (int i = threadIdx.x; i < count * tail; i += ROPE_THREADS) {
                const int k = i / tail, at = tail0 + (i - k * tail) * 8;
                const T *src = x + (size_t)(first + k) * a.xp + at;
                T *dst = y + (size_t)(first + k) * a.yp + at;
#pragma unroll
                for (int b = 0; b < (int)sizeof(T) / 2; ++b) {                    // eight channels: one vector of bf16, two of f32
                    constexpr int N = 16 / sizeof(T);
                    union { uint4 raw; T v[N]; } v;
                    v.raw = reinterpret_cast<const uint4 *>(src)[b];
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (at + b * N + e >= a.c) v.v[e] = from_float<T>(0.f);   // padding channels stay zero
                    reinterpret_cast<uint4 *>(dst)[b] = v.raw;
                }
            }
        } else {
            for (int i = threadIdx.x; i < count * (a.c8 - tail0); i += ROPE_THREADS) {
                const int k = i / (a.c8 - tail0), at = tail0 + i % (a.c8 - tail0);
                y[(size_t)(first + k) * a.yp + at] = at < a.c ? x[(size_t)(first + k) * a.xp + at] : from_float<T>(0.f);
            }
        }
    }
}

template <typename T, int V>
static cudaError_t start_rope(const RopeArgs &a, bool interleaved, int grid, cudaStream_t s)
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
    if (positions && (uintptr_t)positions % 4) DNB_FAIL(DNB_EINVAL, "rope: positions must be 4-byte aligned");
    if (!positions && x->n % d.frames) DNB_FAIL(DNB_EINVAL, "rope: %d images are no whole number of clips of %d frames", x->n, d.frames);
    if ((long long)x->n * x->h >= 1LL << 31) DNB_FAIL(DNB_EUNSUPPORTED, "rope: %d x %d rows", x->n, x->h);
    RopeArgs a;
    memcpy(a.turn, p.turn, sizeof(a.turn));
    memcpy(a.axis, p.axis, sizeof(a.axis));
    a.x = x->data; a.y = y->data; a.positions = positions;
    a.tokens = (long long)x->n * x->h * x->w;
    a.xp = x->cpitch; a.yp = y->cpitch;
    a.c = x->c; a.c8 = round_up(x->c, 8);
    a.h = x->h; a.w = x->w; a.frames = d.frames;
    for (int i = 0; i < 3; ++i) a.origin[i] = d.origin[i];
    a.heads = d.heads; a.head_dim = d.head_dim; a.pairs = p.pairs;
    // the widest vector that the pairs and the heads are whole numbers of
    int v = x->dtype == DNB_BF16 ? 8 : 4;
    while (p.pairs % v || d.head_dim % v) v /= 2;
    // Tokens of a tile: about two items a thread, so that a sine is there for two or more of them; as many as the table holds.
    const int per_token = d.heads * (p.pairs / v);
    int tile = (2 * ROPE_THREADS + per_token - 1) / per_token;
    if (tile > ROPE_TABLE / p.pairs) tile = ROPE_TABLE / p.pairs;
    a.tile = tile;
    const long long tiles = (a.tokens + tile - 1) / tile, cap = (long long)sm_count() * 8;
    const int grid = (int)(tiles < cap ? tiles : cap);
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
            p->turn[i] = turn * 0x1p64L >= 0x1p64L ? 0 : (uint64_t)(turn * 0x1p64L);
            p->axis[i] = (uint8_t)axis;
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
