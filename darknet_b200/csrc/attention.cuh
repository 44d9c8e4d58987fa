// Device code that the cross-attention kernels share.
#pragma once
#include "attention.h"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

namespace dnb {

// What a wait that ran out was for.
enum { AT_QUERIES = 201, AT_SLOT, AT_KEYS, AT_VALUES, AT_SCORES, AT_WEIGHTS, AT_OUTPUT, AT_SMEM_BASE };

// 2^x, as the hardware's one instruction has it (2 ulp); 0 below 2^-126.
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Two floats as three pairs of bf16, each the nearest of what is left.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo)
{
    hi = pack_bf16(x, y);
    x -= __uint_as_float(hi << 16);
    y -= __uint_as_float(hi & 0xffff0000u);
    mid = pack_bf16(x, y);
    x -= __uint_as_float(mid << 16);
    y -= __uint_as_float(mid & 0xffff0000u);
    lo = pack_bf16(x, y);
}

// An MMA whose A lies in TMEM: the weights.  ADD: onto the sums so far, whatever `accumulate` says.
template <bool ADD>
__device__ __forceinline__ void umma_from_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate)
{
    if (ADD)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank)
{
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 at;\n\t"
        "mapa.shared::cluster.u32 at, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [at];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float ld_peer1(uint32_t addr, uint32_t rank)
{
    float v;
    asm volatile("{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %1, %2;\n\tld.shared::cluster.f32 %0, [at];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// Masks of 32 rows, a row a lane, N keys of each, on their way from memory a tile before they are needed: the aligned 16-byte pieces that a row's keys lie
// in, one more than N / 16 since a row may start at any byte, by asynchronous copies that leave out what lies behind the last key.  The bytes in front of
// a row's first are not read.  (Four-byte copies, 17 a warp and tile in place of 5: 300 us in place of 213 for 152 x 256 over 5776 tokens, heads of 64.)
template <int N> struct MaskRows {
    static constexpr int PIECES = N / 16 + 1, BYTES = 32 * PIECES * 16;
};
template <int N>
__device__ __forceinline__ void mask_fetch(uint32_t at, const uint8_t *mask, int key0, int keys, int lane)
{
    constexpr int P = MaskRows<N>::PIECES;
#pragma unroll
    for (int i0 = 0; i0 < 32 * P; i0 += 32) {
        const int i = i0 + lane, row = i / P, piece = i - row * P;
        const uint8_t *p = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mask), row)) + key0;
        const int off = (int)(reinterpret_cast<unsigned long long>(p) & 15u), k = key0 - off + 16 * piece;
        p += 16 * piece - off;
        const uint32_t to = at + 16 * i;
        if (k >= 0) {
            const int n = min(max(keys - k, 0), 16);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "r"(n) : "memory");
        } else {
            uint32_t w[4] = {};
#pragma unroll
            for (int b = 1; b < 16; ++b)
                if (k + b >= 0 && k + b < keys) w[b / 4] |= (uint32_t)p[b] << (b % 4 * 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        }
    }
}
// This lane's row of what mask_fetch brought, a bit a key.
template <int N>
__device__ __forceinline__ void mask_bits(uint32_t at, const uint8_t *mask, int key0, int lane, uint32_t *bits)
{
    constexpr int P = MaskRows<N>::PIECES;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    uint32_t found[P / 2 + 1] = {};
#pragma unroll
    for (int c = 0; c < P; ++c) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + (lane * P + c) * 16) : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (((w[e] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[e]) >> 7 & 0x01010101u;      // a byte of one where there is any bit
        const uint32_t low = __dp4a(w[1], 0x80402010u, __dp4a(w[0], 0x08040201u, 0u)), high = __dp4a(w[3], 0x80402010u, __dp4a(w[2], 0x08040201u, 0u));
        found[c / 2] |= (low | high << 8) << (c % 2 * 16);
    }
    const uint32_t off = (uint32_t)((reinterpret_cast<unsigned long long>(mask) + key0) & 15u);
#pragma unroll
    for (int c = 0; c < N / 32; ++c) bits[c] = __funnelshift_r(found[c], found[c + 1], off);
    __syncwarp();                                                       // every lane has read: the next tile's may come
}

// The keys that CTA `rank` of `splits` walks over, in tiles of `size`: [first, first + count) of an image's `keys`.
__device__ __forceinline__ void share_of_keys(int keys, int size, int rank, int splits, int &first, int &count)
{
    const int all = (keys + size - 1) / size, per = (all + splits - 1) / splits;
    first = min(rank * per, all);
    count = min(first + per, all) - first;
}

// Joins the rows that the CTAs of a cluster hold of the same queries: in every CTA, at the same addresses of shared memory, row r's sum of weighted
// values at rows + r * pitch floats, its largest scaled score (log2) in tops[r] and its sum of weights in sums[r] (0: its row holds nothing).
// Four channels an item, the items dealt out over the cluster's threads; the additions in the order of the ranks, which is the keys'.  All of an item's
// loads are on their way before the first is used: one trip to the neighbours, not one a neighbour.  N: the CTAs, rounded up to 2, 4 or 8.
// out(r): where row r's d channels go, or null.
template <typename T, int N, typename Out>
__device__ __forceinline__ void join_rows_of(uint32_t rows, int pitch, uint32_t tops, uint32_t sums, int count, int d, int rank, int splits, int tid, int threads, Out out)
{
    const int chunks = d / 4;
    for (int i = tid * splits + rank; i < count * chunks; i += threads * splits) {
        const int r = i / chunks, c = (i - r * chunks) * 4;
        T *to = out(r);
        if (!to) continue;
        float top[N], weight[N];
        float4 x[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t from = k < splits ? k : 0;
            top[k] = ld_peer1(tops + 4 * r, from);
            weight[k] = ld_peer1(sums + 4 * r, from);
            x[k] = ld_peer(rows + (r * pitch + c) * 4, from);
        }
        float most = -INFINITY, total = 0.f;
#pragma unroll
        for (int k = 0; k < N; ++k) most = fmaxf(most, top[k]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const bool has = k < splits && weight[k] != 0.f;
            const float w = top[k] == most ? 1.f : ex2(top[k] - most);
            total = has ? fmaf(weight[k], w, total) : total;
            o.x = has ? fmaf(x[k].x, w, o.x) : o.x;
            o.y = has ? fmaf(x[k].y, w, o.y) : o.y;
            o.z = has ? fmaf(x[k].z, w, o.z) : o.z;
            o.w = has ? fmaf(x[k].w, w, o.w) : o.w;
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2 *>(to + c) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
        else *reinterpret_cast<float4 *>(to + c) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}
template <typename T, typename Out>
__device__ __forceinline__ void join_rows(uint32_t rows, int pitch, uint32_t tops, uint32_t sums, int count, int d, int rank, int splits, int tid, int threads, Out out)
{
    if (splits <= 2) join_rows_of<T, 2>(rows, pitch, tops, sums, count, d, rank, splits, tid, threads, out);
    else if (splits <= 4) join_rows_of<T, 4>(rows, pitch, tops, sums, count, d, rank, splits, tid, threads, out);
    else join_rows_of<T, 8>(rows, pitch, tops, sums, count, d, rank, splits, tid, threads, out);
}

}  // namespace dnb
