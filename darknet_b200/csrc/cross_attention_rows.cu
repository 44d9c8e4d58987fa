// Cross attention for few query rows a key head: single tokens, and the query heads that share its keys.
//
// The bytes of keys and values bound it: each is read once, by TMA, through a ring of tiles of 64 keys that keeps about 100 KB an SM's block (two of
// them an SM) on the way.  Four warps, 16 keys of a tile each, multiply them by up to 16 rows with mma.sync: the 128 rows of a tcgen05 product would be
// empty but for a few, its TMEM round trip is a latency for each tile, and the arithmetic is far from any bound either way.  A warp has a running maximum
// and sum of its own keys; warps, and the CTAs of a cluster that share the keys of one head, meet once at the end.
// Measured: 32 tokens over 5776 keys, 16 heads over 4 of 128: 61 us in bf16 (6.2 TB/s), 153 in f32 (5.0 TB/s); one token over 361 keys, 8 heads of 64: 5.9 us back to back.
//
// f32 operands are sums of three bf16 numbers (24 bits of mantissa), their product the six products of parts that reach 2^-24 of it, smallest first; a tile's
// sums are added to the rows' in fp32, since the tensor cores' sums lose a little at each addition.  A lane reads four channels of a key at once: which
// channel of the head stands where along a product's K, and which key or channel along its N, is free as long as both operands agree, and is chosen
// such that the eight lanes of a 16-byte load meet all banks.
#include <atomic>

#include "attention.cuh"

namespace dnb {

int encode_tensor_map(CUtensorMap *map, int elem_kind, int rank, void *base, const uint64_t *dims, const uint64_t *strides_bytes, const uint32_t *box, int swizzle_bytes);

namespace {

constexpr int R_KEYS = 64, R_WARPS = 4, R_THREADS = R_WARPS * 32 + 32;
constexpr float R_MOVE = 8.f;                     // how far (log2) scores may outgrow the running maximum before the sums are corrected

template <typename T, int DP> struct RowsCfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int BOX_CHANNELS = 128 / sizeof(T), BOXES = DP / BOX_CHANNELS;
    static constexpr uint32_t BOX = R_KEYS * 128, TILE = BOXES * BOX;
    static constexpr int STAGES = 12 / BOXES;
    static constexpr int PITCH = DP + 4;
    static constexpr uint32_t WORK = STAGES * TILE, Q_PART = DP / 16 * 512;    // Q_PART: fragments of one part of the queries, f32 only
    static constexpr uint32_t BYTES = WORK + (F32 ? 3 * Q_PART : 0);           // in front of RowsShared
    static_assert((R_WARPS + 1) * 16 * PITCH * 4 <= (int)WORK, "the warps' sums fit where the tiles were");
};

struct RowsShared {
    uint64_t full[12], empty[12];
    int abort_flag;
    float top[R_WARPS * 16], sum[R_WARPS * 16], all_top[16], all_sum[16];
};

struct alignas(64) RowsArgs {
    CUtensorMap tmk, tmv;
    AttnArgs a;
    int splits;
    float scale_log2;
};

__device__ __forceinline__ void ldsm4(uint32_t at, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t at, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(R_THREADS, 2)
attention_rows_kernel(const __grid_constant__ RowsArgs t)
{
    using C = RowsCfg<T, DP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const AttnArgs &a = t.a;
    const uint32_t ring = smem_u32(smem_raw);
    if (ring & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, AT_SMEM_BASE);
        return;
    }
    RowsShared *sh = reinterpret_cast<RowsShared *>(smem_raw + C::BYTES);
    volatile int *abort_flag = &sh->abort_flag;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = (int)(blockIdx.x % (unsigned)t.splits), job = (int)(blockIdx.x / (unsigned)t.splits);
    const int kv_head = job % a.kv_heads, image = job / a.kv_heads;
    const int rows = a.lq * a.group;                                    // row r: token r / group, head r % group of the group
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(smem_u32(&sh->full[i]), 1);
            mbar_init(smem_u32(&sh->empty[i]), R_WARPS);
        }
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    grid_dependency_wait();
    launch_dependents_if_small();

    int keys = a.lk, first, tiles;
    if (a.lengths) keys = min(max(a.lengths[image], 0), a.lk);
    share_of_keys(keys, R_KEYS, rank, t.splits, first, tiles);
    const int boxes = C::F32 ? (a.d + C::BOX_CHANNELS - 1) / C::BOX_CHANNELS : C::BOXES;     // that hold channels of the head
    // the token and head of row r: where its channels start in q (and, with y's pitch, in y)
    auto q_at = [&](int r, int pitch) { return ((size_t)image * a.lq + r / a.group) * pitch + (kv_head * a.group + r % a.group) * a.d; };

    if (warp == R_WARPS) {
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; i < 2 * tiles; ++i) {
            const uint32_t full = smem_u32(&sh->full[stage]);
            if (!mbar_wait_known(smem_u32(&sh->empty[stage]), phase ^ 1, abort_flag, a.status, AT_SLOT, a.polls) || gave_up(abort_flag)) break;
            if (elect_one() && !(a.debug & 32 && i == 1)) {
                mbar_expect_tx(full, boxes * C::BOX);
                for (int b = 0; b < boxes; ++b)
                    tma_load_4d(ring + stage * C::TILE + b * C::BOX, i & 1 ? &t.tmv : &t.tmk, full, b * C::BOX_CHANNELS, kv_head, (first + i / 2) * R_KEYS, a.kn == 1 ? 0 : image);
            }
            if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
        }
        __syncwarp();
    }

    const int g = lane >> 2, c2 = (lane & 3) * 2;                       // this lane's rows g and g + 8 of a product, columns c2 and c2 + 1
    float o[DP / 8][4] = {}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    const uint4 *q_parts = reinterpret_cast<const uint4 *>(smem_raw + C::WORK) + lane;
    if (warp < R_WARPS && tiles > 0) {
        if constexpr (C::F32) {
            // the queries' fragments in three parts, the same for every warp: along K, channels 4 t .. 4 t + 3 of 16 stand at 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (t = lane % 4)
            for (int i = warp; i < DP / 16; i += R_WARPS) {
                float4 x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = g + e * 8, c = i * 16 + 2 * c2;
                    x[e] = r < rows && c < a.d ? *reinterpret_cast<const float4 *>((const float *)a.q + q_at(r, a.qp) + c) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                uint4 f[3];
                split2(x[0].x, x[0].y, f[0].x, f[1].x, f[2].x);
                split2(x[1].x, x[1].y, f[0].y, f[1].y, f[2].y);
                split2(x[0].z, x[0].w, f[0].z, f[1].z, f[2].z);
                split2(x[1].z, x[1].w, f[0].w, f[1].w, f[2].w);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4 *>(smem_raw + C::WORK + p * C::Q_PART + i * 512 + lane * 16) = f[p];
            }
            asm volatile("bar.sync 1, %0;" ::"n"(R_WARPS * 32) : "memory");     // not with the warp that loads
        }
        uint32_t q[C::F32 ? 1 : DP / 16][4];
        if constexpr (!C::F32)
#pragma unroll
            for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = g + (e & 1) * 8, c = i * 16 + c2 + (e >> 1) * 8;
                    q[i][e] = r < rows && c < a.d ? *reinterpret_cast<const uint32_t *>((const __nv_bfloat16 *)a.q + q_at(r, a.qp) + c) : 0u;
                }
        const uint8_t *mask[2] = {nullptr, nullptr};
        if (a.mask)
            for (int e = 0; e < 2; ++e) mask[e] = a.mask + (long long)image * a.mask_image + (long long)(g + e * 8 < rows ? (g + e * 8) / a.group : 0) * a.mask_query;
        const int m = lane >> 3, mr = lane & 7;                         // the 8x8 matrix and its row whose address this lane gives
        int stage = 0;
        uint32_t phase = 0;
        auto next = [&]() { if (++stage == C::STAGES) { stage = 0; phase ^= 1; } };
        for (int j = 0; j < tiles; ++j) {
            const int key0 = (first + j) * R_KEYS + warp * 16, left = keys - key0;
            bool in[2][4];                                              // row e, keys c2, c2 + 1, 8 + c2, 8 + c2 + 1; of f32: t, t + 4, t + 8, t + 12
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = C::F32 ? (lane & 3) + 4 * i : (i >> 1) * 8 + c2 + (i & 1);
                    in[e][i] = key < left && (!a.mask || mask[e][key0 + key]);
                }
            mbar_wait_tight(smem_u32(&sh->full[stage]), phase, abort_flag, a.status, AT_KEYS, a.polls);
            float s[2][4] = {};
            if constexpr (C::F32) {
                // keys along N: n is key (n & 1) * 4 + n / 2 of eight
                const uint8_t *at = smem_raw + stage * C::TILE + (warp * 16 + (g & 1) * 4 + (g >> 1)) * 128;
                const int turn = ((g & 1) * 4 + (g >> 1)) << 4;         // the swizzle of that row
                float small[2][4] = {};                                 // the products of parts but the highest
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    if (i * 16 >= a.d) break;
                    uint32_t f[3][4];
#pragma unroll
                    for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4 *>(f[p]) = q_parts[p * (C::Q_PART / 16) + i * 32];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float4 x = *reinterpret_cast<const float4 *>(at + (i >> 1) * C::BOX + n * 1024 + (((i & 1) * 64 + (lane & 3) * 16) ^ turn));
                        uint32_t b[3][2];
                        split2(x.x, x.y, b[0][0], b[1][0], b[2][0]);
                        split2(x.z, x.w, b[0][1], b[1][1], b[2][1]);
                        mma16816(small[n], f[2], b[0][0], b[0][1]);
                        mma16816(small[n], f[0], b[2][0], b[2][1]);
                        mma16816(small[n], f[1], b[1][0], b[1][1]);
                        mma16816(small[n], f[1], b[0][0], b[0][1]);
                        mma16816(small[n], f[0], b[1][0], b[1][1]);
                        mma16816(s[n], f[0], b[0][0], b[0][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] += small[n][e];
            } else {
                const int key = warp * 16 + (m >> 1) * 8 + mr;
                const uint32_t at = ring + stage * C::TILE + key * 128;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    const int c = i * 16 + (m & 1) * 8;
                    uint32_t b[4];
                    ldsm4(at + (c >> 6) * C::BOX + (((c & 63) * 2) ^ (mr << 4)), b);
                    mma16816(s[0], q[i], b[0], b[1]);
                    mma16816(s[1], q[i], b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->empty[stage]));
            next();
            float grown[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                grown[e] = top[e];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float &v = s[i >> 1][e * 2 + (i & 1)];
                    v = in[e][i] ? v * t.scale_log2 : -INFINITY;
                    grown[e] = fmaxf(grown[e], v);
                }
                grown[e] = fmaxf(grown[e], __shfl_xor_sync(0xffffffffu, grown[e], 1));
                grown[e] = fmaxf(grown[e], __shfl_xor_sync(0xffffffffu, grown[e], 2));
            }
            if (__any_sync(0xffffffffu, grown[0] - top[0] > R_MOVE || grown[1] - top[1] > R_MOVE)) {
                float shrink[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    shrink[e] = grown[e] == top[e] ? 1.f : ex2(top[e] - grown[e]);
                    top[e] = grown[e];
                    sum[e] *= shrink[e];
                }
#pragma unroll
                for (int i = 0; i < DP / 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] *= shrink[e >> 1];
            }
            uint32_t p[C::F32 ? 3 : 1][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = top[e] == -INFINITY ? 0.f : top[e];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = ex2(s[i][e * 2] - base), z = ex2(s[i][e * 2 + 1] - base);
                    sum[e] += x + z;
                    if constexpr (C::F32) split2(x, z, p[0][i * 2 + e], p[1][i * 2 + e], p[2][i * 2 + e]);
                    else p[0][i * 2 + e] = pack_bf16(x, z);
                }
            }
            mbar_wait_tight(smem_u32(&sh->full[stage]), phase, abort_flag, a.status, AT_VALUES, a.polls);
            const uint32_t v_tile = stage * C::TILE;
            if ((left < 16 && keys < a.lk) || (a.mask && a.mask_query == 0)) {
                // values that no weight reaches may be anything: zeros in their place, this warp's keys by this warp
                const int key = lane >> 1;
                if (key >= left || (a.mask && a.mask_query == 0 && !mask[0][key0 + key])) {
#pragma unroll
                    for (int b = 0; b < C::BOXES; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<uint4 *>(smem_raw + v_tile + b * C::BOX + (warp * 16 + key) * 128 + (lane & 1) * 64 + e * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();                                     // before the slot's next load
                __syncwarp();
            }
            if constexpr (C::F32) {
                // channels along N: of a box of 32, product e's n is channel 4 * ((n & 1) * 4 + n / 2) + e
                const uint8_t *at = smem_raw + v_tile + (warp * 16 + (lane & 3)) * 128;
                const int chunk = ((g & 1) * 4 + (g >> 1)) ^ (lane & 3);  // keys t + 4 and t + 12: the chunk four further
#pragma unroll
                for (int b = 0; b < C::BOXES; ++b) {
                    if (b * 32 >= a.d) break;
                    float x[4][4];                                      // keys t, t + 4, t + 8, t + 12
#pragma unroll
                    for (int k = 0; k < 4; ++k) *reinterpret_cast<float4 *>(x[k]) = *reinterpret_cast<const float4 *>(at + b * C::BOX + k * 512 + ((chunk ^ (k & 1) * 4) << 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t w[3][2];
                        split2(x[0][e], x[1][e], w[0][0], w[1][0], w[2][0]);
                        split2(x[2][e], x[3][e], w[0][1], w[1][1], w[2][1]);
                        float now[4] = {};
                        mma16816(now, p[2], w[0][0], w[0][1]);
                        mma16816(now, p[0], w[2][0], w[2][1]);
                        mma16816(now, p[1], w[1][0], w[1][1]);
                        mma16816(now, p[1], w[0][0], w[0][1]);
                        mma16816(now, p[0], w[1][0], w[1][1]);
                        mma16816(now, p[0], w[0][0], w[0][1]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[b * 4 + e][k] += now[k];
                    }
                }
            } else {
                const int key = warp * 16 + (m & 1) * 8 + mr;
                const uint32_t at = ring + v_tile + key * 128;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    const int c = i * 16 + (m >> 1) * 8;
                    uint32_t b[4];
                    ldsm4t(at + (c >> 6) * C::BOX + (((c & 63) * 2) ^ (mr << 4)), b);
                    mma16816(o[2 * i], p[0], b[0], b[1]);
                    mma16816(o[2 * i + 1], p[0], b[2], b[3]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->empty[stage]));
            next();
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
    }
    __syncthreads();                                                    // every tile has been read: its memory takes the sums
    float *parts = reinterpret_cast<float *>(smem_raw), *whole = parts + R_WARPS * 16 * C::PITCH;
    if (warp < R_WARPS) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = warp * 16 + g + e * 8;
            if ((lane & 3) == 0) { sh->top[r] = top[e]; sh->sum[r] = sum[e]; }
            if (g + e * 8 >= rows) continue;
            if constexpr (C::F32) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        *reinterpret_cast<float4 *>(parts + r * C::PITCH + i * 32 + k * 16 + 2 * c2) =
                            make_float4(o[4 * i][e * 2 + k], o[4 * i + 1][e * 2 + k], o[4 * i + 2][e * 2 + k], o[4 * i + 3][e * 2 + k]);
            } else
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) *reinterpret_cast<float2 *>(parts + r * C::PITCH + i * 8 + c2) = make_float2(o[i][e * 2], o[i][e * 2 + 1]);
        }
    }
    __syncthreads();
    // the warps' sums to the block's, or to the output where the block has all keys
    const int chunks = a.d / 4;
    for (int i = tid; i < rows * chunks && !*abort_flag; i += R_THREADS) {
        const int r = i / chunks, c = (i - r * chunks) * 4;
        float most = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < R_WARPS; ++w) most = fmaxf(most, sh->top[w * 16 + r]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < R_WARPS; ++w) {
            const float l = sh->sum[w * 16 + r], m = sh->top[w * 16 + r];
            if (l == 0.f) continue;
            const float f = m == most ? 1.f : ex2(m - most);
            const float4 z = *reinterpret_cast<const float4 *>(parts + (w * 16 + r) * C::PITCH + c);
            total += l * f;
            x.x = fmaf(z.x, f, x.x); x.y = fmaf(z.y, f, x.y); x.z = fmaf(z.z, f, x.z); x.w = fmaf(z.w, f, x.w);
        }
        if (t.splits == 1) {
            const float inv = total == 0.f ? 0.f : 1.f / total;
            if constexpr (C::F32) *reinterpret_cast<float4 *>((float *)a.y + q_at(r, a.yp) + c) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            else *reinterpret_cast<uint2 *>((__nv_bfloat16 *)a.y + q_at(r, a.yp) + c) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        } else {
            *reinterpret_cast<float4 *>(whole + r * C::PITCH + c) = x;
            if (c == 0) { sh->all_top[r] = most; sh->all_sum[r] = total; }
        }
    }
    if (t.splits > 1) {
        __syncwarp();
        cluster_sync_all();
        if (!*abort_flag)
            join_rows<T>(smem_u32(whole), C::PITCH, smem_u32(sh->all_top), smem_u32(sh->all_sum), rows, a.d, rank, t.splits, tid, R_THREADS,
                                     [&](int r) { return (T *)a.y + q_at(r, a.yp); });
        __syncwarp();
        cluster_sync_all();
    }
    if (*abort_flag) {                                                  // loads in flight land before their memory goes
        const long long begin = clock64();
        while (clock64() - begin < 4000000LL) { }
    }
}

typedef void (*RowsKernel)(RowsArgs);
struct RowsVariant {
    RowsKernel kernel;
    size_t bytes;
};
template <typename T, int DP> RowsVariant rows_variant() { return {attention_rows_kernel<T, DP>, RowsCfg<T, DP>::BYTES + sizeof(RowsShared)}; }

}  // namespace

// Up to the 16 rows of its one product.  us of this kernel / of the one for 128 rows at 16 rows, which costs that one what one row or 128 do (8 key heads):
//   4 images of 5776 keys, heads of 64  bf16 13.9 / 20.3  f32 28.5 / 51.1     heads of 128  bf16 23.4 / 27.5  f32 49.6 / 110
//   8 of 1444                           bf16 10.3 / 13.2  f32 17.0 / 29.9                   bf16 15.1 / 17.1  f32 29.4 / 62.5
//   1 of 361                            bf16  6.6 / 6.7   f32  6.1 / 10.7                   bf16 10.1 / 8.3   f32  9.4 / 18.4   (at 8 rows bf16 7.7 / 8.3)
// A second product of 16 rows, for up to 32, is not there: from 17 rows on the right-hand figures hold.
bool attention_rows_covers(const AttnArgs &a)
{
    return a.d <= 128 && (long long)a.lq * a.group <= 16 && (long long)a.n * a.kv_heads < 1LL << 28;
}

int launch_attention_rows(const AttnArgs &a, int dtype, cudaStream_t stream)
{
    const bool f32 = dtype == DNB_F32, big = a.d > 64;
    const uint64_t es = f32 ? 4 : 2;
    RowsArgs t;
    t.a = a;
    t.scale_log2 = a.scale * 1.4426950408889634f;
    auto map = [&](CUtensorMap *m, const void *data, int pitch) {
        const uint64_t dims[4] = {(uint64_t)a.d, (uint64_t)a.kv_heads, (uint64_t)a.lk, (uint64_t)a.kn};
        const uint64_t strides[3] = {a.d * es, pitch * es, (uint64_t)a.lk * pitch * es};
        const uint32_t box[4] = {f32 ? 32u : 64u, 1, R_KEYS, 1};
        return encode_tensor_map(m, f32 ? 0 : 1, 4, const_cast<void *>(data), dims, strides, box, 128);
    };
    DNB_TRY(map(&t.tmk, a.k, a.kp));
    DNB_TRY(map(&t.tmv, a.v, a.vp));
    // Two blocks an SM: the keys over as many of them as there is room for.  One token, us over 1 / 2 / 4 / 8 blocks a head: 8 heads of 64, 361 keys
    // 6.6 / 6.1 / 6.1 / 5.8 (f32 11.0 / 8.0 / 7.0 / 5.7), 1444 keys 14.7 / 10.6 / 7.6 / 6.6; 80 heads over 1 / 2 / 3 / 4 15.1 / 11.3 / 9.7 / 16.0.
    const long long jobs = (long long)a.n * a.kv_heads;
    const int key_tiles = (a.lk + R_KEYS - 1) / R_KEYS;
    const long long room = 2LL * sm_count() / jobs;
    t.splits = room < 2 ? 1 : (int)(room < 8 ? room : 8);
    // f32 images of lengths of their own: twice the blocks while each keeps twelve tiles, so that a short image's place is taken by a long one's keys
    // (32 tokens over maps of up to 5776, 4 key heads of 128: 127 us, from 145; bf16 46 either way).
    if (f32 && a.lengths)
        while (t.splits < 8 && (t.splits + 1) * jobs <= 4LL * sm_count() && key_tiles >= 12 * (t.splits + 1)) ++t.splits;
    if (t.splits > key_tiles) t.splits = key_tiles;
    const RowsVariant kern = f32 ? (big ? rows_variant<float, 128>() : rows_variant<float, 64>())
                                 : (big ? rows_variant<__nv_bfloat16, 128>() : rows_variant<__nv_bfloat16, 64>());
    static std::atomic<bool> done[64][4];
    int dev = 0;
    DNB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) DNB_FAIL(DNB_ECUDA, "attention: device %d", dev);
    if (!done[dev][2 * f32 + big].load(std::memory_order_acquire)) {
        DNB_CUDA(cudaFuncSetAttribute(kern.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kern.bytes));
        done[dev][2 * f32 + big].store(true, std::memory_order_release);
    }
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = pdl_enabled() && jobs * t.splits <= EARLY_BLOCKS ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)t.splits; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(jobs * t.splits));
    cfg.blockDim = dim3(R_THREADS);
    cfg.dynamicSmemBytes = kern.bytes;
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    DNB_CUDA(cudaLaunchKernelEx(&cfg, kern.kernel, t));
    DNB_LAUNCH_CHECK("attention");
    return DNB_OK;
}

}  // namespace dnb
