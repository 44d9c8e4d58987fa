// Cross attention of f32 tensors: fp32 products and sums on the CUDA cores.
//
// A block of 256 threads holds 16 R query rows (a row: one query token of one head; heads that share keys lie side by side) and walks over the keys 64 at a time;
// a thread holds R rows by 4 keys of the scores and R rows by DT / 16 channels of the output, the 16 threads of a row meet in shuffles.  The next tile of
// keys travels (cp.async) while the weights meet the values, the values while the scores are made.  The FMAs bound it: 4 d of them a row and four keys,
// against R + 4 sixteen-byte loads from shared memory for R * 16 of the first product.  R = 1 serves single tokens, whose bytes bound them.
// Few rows: the keys are split over the CTAs of a cluster, which join their sums through distributed shared memory.
#include <atomic>

#include "attention.cuh"

namespace dnb {
namespace {

constexpr int F_KEYS = 64, F_THREADS = 256;

template <int DT, int R> struct F32Cfg {
    static constexpr int ROWS = 16 * R, PITCH = DT + 4, P_PITCH = F_KEYS + 4;
    static constexpr int K_AT = ROWS * PITCH, V_AT = K_AT + F_KEYS * PITCH, P_AT = V_AT + F_KEYS * PITCH, TOP_AT = P_AT + ROWS * P_PITCH, SUM_AT = TOP_AT + ROWS;
    static constexpr int BYTES = (SUM_AT + ROWS) * 4;
};

struct F32Args {
    AttnArgs a;
    int q_tokens, q_tiles, splits;
    float scale_log2;
};

// DT: channels of a head as they lie in shared memory (32, 64 or 128), behind d zeros.
template <int DT, int R>
__global__ void __launch_bounds__(F_THREADS)
attention_f32_kernel(const __grid_constant__ F32Args t)
{
    using C = F32Cfg<DT, R>;
    constexpr int COLS = DT / 16, VW = COLS < 4 ? COLS : 4, VN = COLS / VW;   // a thread's channels: VN pieces of VW, 16 * VW apart
    extern __shared__ __align__(16) float sm[];
    const AttnArgs &a = t.a;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int rank = (int)(blockIdx.x % (unsigned)t.splits), job = (int)(blockIdx.x / (unsigned)t.splits);
    const int q_tile = job % t.q_tiles, kv_head = job / t.q_tiles % a.kv_heads, image = job / t.q_tiles / a.kv_heads;
    const int token0 = q_tile * t.q_tokens, rows_here = min(t.q_tokens, a.lq - token0) * a.group;
    grid_dependency_wait();
    launch_dependents_if_small();

    int keys = a.lk, first, tiles;
    if (a.lengths) keys = min(max(a.lengths[image], 0), a.lk);
    share_of_keys(keys, F_KEYS, rank, t.splits, first, tiles);
    const int end = min(keys, (first + tiles) * F_KEYS);
    const uint8_t *mask = a.mask ? a.mask + (long long)image * a.mask_image : nullptr;
    const size_t base = (size_t)(a.kn == 1 ? 0 : image) * a.lk;
    const float *k = (const float *)a.k + base * a.kp + kv_head * a.d, *v = (const float *)a.v + base * a.vp + kv_head * a.d;

    // 64 rows of keys or values from key0 on; zeros where there is none, or none that any query sees
    auto load = [&](const float *src, int pitch, int at, int key0) {
        for (int i = tid; i < F_KEYS * DT / 4; i += F_THREADS) {
            const int r = i / (DT / 4), c = i % (DT / 4) * 4, key = key0 + r;
            const bool in = key < end && c < a.d && !(mask && a.mask_query == 0 && !mask[key]);
            cp_async16(smem_u32(sm + at + r * C::PITCH + c), in ? src + (size_t)key * pitch + c : src, in);
        }
        cp_async_commit();
    };
    if (tiles > 0) {
        for (int i = tid; i < C::ROWS * DT / 4; i += F_THREADS) {
            const int r = i / (DT / 4), c = i % (DT / 4) * 4;
            const bool in = r < rows_here && c < a.d;
            const float *src = (const float *)a.q + ((size_t)image * a.lq + token0 + (in ? r / a.group : 0)) * a.qp + (kv_head * a.group + (in ? r % a.group : 0)) * a.d + (in ? c : 0);
            cp_async16(smem_u32(sm + r * C::PITCH + c), src, in);
        }
        load(k, a.kp, C::K_AT, first * F_KEYS);
        load(v, a.vp, C::V_AT, first * F_KEYS);
    }

    float o[R][COLS] = {}, top[R], sum[R] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) top[r] = -INFINITY;
    for (int j = 0; j < tiles; ++j) {
        const int key0 = (first + j) * F_KEYS;
        cp_async_wait<1>();                                   // the keys; the values may be under way
        __syncthreads();
        float s[R][4] = {};
#pragma unroll 4
        for (int c = 0; c < DT; c += 4) {
            float4 q4[R], k4[4];
#pragma unroll
            for (int r = 0; r < R; ++r) q4[r] = *reinterpret_cast<const float4 *>(sm + (ty * R + r) * C::PITCH + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) k4[i] = *reinterpret_cast<const float4 *>(sm + C::K_AT + (tx + 16 * i) * C::PITCH + c);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[r][i] = fmaf(q4[r].w, k4[i].w, fmaf(q4[r].z, k4[i].z, fmaf(q4[r].y, k4[i].y, fmaf(q4[r].x, k4[i].x, s[r][i]))));
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = ty * R + r;
            const uint8_t *seen = mask ? mask + (long long)(token0 + (row < rows_here ? row / a.group : 0)) * a.mask_query : nullptr;
            float most = top[r];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = key0 + tx + 16 * i;
                s[r][i] = key < end && (!seen || seen[key]) ? s[r][i] * t.scale_log2 : -INFINITY;
                most = fmaxf(most, s[r][i]);
            }
#pragma unroll
            for (int x = 8; x; x >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
            const float from = most == -INFINITY ? 0.f : most, shrink = most == top[r] ? 1.f : ex2(top[r] - most);
            top[r] = most;
            sum[r] *= shrink;
#pragma unroll
            for (int c = 0; c < COLS; ++c) o[r][c] *= shrink;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = ex2(s[r][i] - from);
                sum[r] += p;
                sm[C::P_AT + row * C::P_PITCH + tx + 16 * i] = p;
            }
        }
        __syncthreads();                                      // the weights are there, and the keys have been read
        if (j + 1 < tiles) load(k, a.kp, C::K_AT, key0 + F_KEYS);
        if (j + 1 < tiles) cp_async_wait<1>();                // the values
        else cp_async_wait<0>();
        __syncthreads();
#pragma unroll 2
        for (int i = 0; i < F_KEYS; i += 4) {
            float4 p4[R];
#pragma unroll
            for (int r = 0; r < R; ++r) p4[r] = *reinterpret_cast<const float4 *>(sm + C::P_AT + (ty * R + r) * C::P_PITCH + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float vv[COLS];
#pragma unroll
                for (int n = 0; n < VN; ++n) {
                    const float *at = sm + C::V_AT + (i + e) * C::PITCH + n * 16 * VW + tx * VW;
                    if constexpr (VW == 4) *reinterpret_cast<float4 *>(vv + n * VW) = *reinterpret_cast<const float4 *>(at);
                    else *reinterpret_cast<float2 *>(vv + n * VW) = *reinterpret_cast<const float2 *>(at);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float p = e == 0 ? p4[r].x : e == 1 ? p4[r].y : e == 2 ? p4[r].z : p4[r].w;
#pragma unroll
                    for (int c = 0; c < COLS; ++c) o[r][c] = fmaf(p, vv[c], o[r][c]);
                }
            }
        }
        __syncthreads();                                      // weights and values have been read
        if (j + 1 < tiles) load(v, a.vp, C::V_AT, key0 + F_KEYS);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int x = 8; x; x >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);

    auto out = [&](int row) -> float * {
        return row >= rows_here ? nullptr : (float *)a.y + ((size_t)image * a.lq + token0 + row / a.group) * a.yp + (kv_head * a.group + row % a.group) * a.d;
    };
    if (t.splits == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float *y = out(ty * R + r);
            const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];
            if (y)
#pragma unroll
                for (int n = 0; n < VN; ++n) {
                    const int c = n * 16 * VW + tx * VW;
                    if (c >= a.d) continue;                   // d is a multiple of 8, a piece 2 or 4
                    if constexpr (VW == 4)
                        *reinterpret_cast<float4 *>(y + c) = make_float4(o[r][n * VW] * inv, o[r][n * VW + 1] * inv, o[r][n * VW + 2] * inv, o[r][n * VW + 3] * inv);
                    else
                        *reinterpret_cast<float2 *>(y + c) = make_float2(o[r][n * VW] * inv, o[r][n * VW + 1] * inv);
                }
        }
        return;
    }
    __syncthreads();                                          // the queries' rows become the sums'
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = ty * R + r;
        if (tx == 0) { sm[C::TOP_AT + row] = top[r]; sm[C::SUM_AT + row] = sum[r]; }
#pragma unroll
        for (int n = 0; n < VN; ++n)
#pragma unroll
            for (int e = 0; e < VW; ++e) sm[row * C::PITCH + n * 16 * VW + tx * VW + e] = o[r][n * VW + e];
    }
    cluster_sync_all();
    join_rows<float>(smem_u32(sm), C::PITCH, smem_u32(sm + C::TOP_AT), smem_u32(sm + C::SUM_AT), min(rows_here, C::ROWS), a.d, rank, t.splits, tid, F_THREADS, out);
    cluster_sync_all();
}

typedef void (*F32Kernel)(F32Args);
template <int DT> F32Kernel f32_kernel(int r) { return r == 1 ? attention_f32_kernel<DT, 1> : attention_f32_kernel<DT, 4>; }
template <int DT> int f32_bytes(int r) { return r == 1 ? F32Cfg<DT, 1>::BYTES : F32Cfg<DT, 4>::BYTES; }

}  // namespace

bool attention_f32_covers(const AttnArgs &a, int dtype)
{
    return dtype == DNB_F32 && a.d <= 128 && a.group <= 64 && (long long)a.n * a.kv_heads * a.lq < 1LL << 28;
}

int launch_attention_f32(const AttnArgs &a, cudaStream_t stream)
{
    F32Args t;
    t.a = a;
    const int r = (long long)a.lq * a.group <= 16 ? 1 : 4, dt = a.d <= 32 ? 0 : a.d <= 64 ? 1 : 2;
    t.q_tokens = 16 * r / a.group;
    t.q_tiles = (a.lq + t.q_tokens - 1) / t.q_tokens;
    t.scale_log2 = a.scale * 1.4426950408889634f;
    const F32Kernel kern = dt == 0 ? f32_kernel<32>(r) : dt == 1 ? f32_kernel<64>(r) : f32_kernel<128>(r);
    const int bytes = dt == 0 ? f32_bytes<32>(r) : dt == 1 ? f32_bytes<64>(r) : f32_bytes<128>(r);
    static std::atomic<bool> done[64][6];
    int dev = 0;
    DNB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) DNB_FAIL(DNB_ECUDA, "attention: device %d", dev);
    std::atomic<bool> &ready = done[dev][dt * 2 + (r == 1)];
    if (!ready.load(std::memory_order_acquire)) {
        DNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        ready.store(true, std::memory_order_release);
    }
    const long long jobs = (long long)a.n * a.kv_heads * t.q_tiles;
    const int key_tiles = (a.lk + F_KEYS - 1) / F_KEYS, room = sm_count() * (dt == 2 ? 1 : dt == 1 ? 3 : 4);
    t.splits = 1;
    while (t.splits < 8 && jobs * t.splits * 2 <= room && key_tiles >= t.splits * 4) t.splits *= 2;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = pdl_enabled() && jobs * t.splits <= EARLY_BLOCKS ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)t.splits; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(jobs * t.splits));
    cfg.blockDim = dim3(F_THREADS);
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    DNB_CUDA(cudaLaunchKernelEx(&cfg, kern, t));
    DNB_LAUNCH_CHECK("attention");
    return DNB_OK;
}

}  // namespace dnb
