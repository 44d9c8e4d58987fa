// Cross attention of f32 tensors on the tensor cores: every operand as the sum of three bf16 numbers (24 bits of mantissa in all), a product of two of them
// as the six products of parts that reach 2^-24 of it, smallest first.
//
//   S = Q K^T     six tcgen05.mma a step of 16 channels, S in TMEM
//   P = exp2(S * scale * log2 e - m), in three parts
//   O = O + P V   six a step of 16 keys; a tile of 64 keys has its own sum in TMEM, and O itself stays in registers: the tensor cores' sums lose a little at
//                 each addition, which over 64 keys stays below what fp32 sums of that length lose, and over thousands would not
//
// A CTA holds 128 query rows (a row: one query token of one head; heads that share keys lie side by side) and walks over the keys 64 at a time: eight warps make
// the weights (half a row a thread) and add the tiles up, four split the keys into parts, four the values, one issues the products.  S and P have two places
// each, so that a tile's scores are made while the tile before is weighed.  A tile's chain of hand-overs bounds it, 1.9 us of 64 keys and heads of 64 (the
// products alone would take 0.8), 4.6 of heads of 128, whose keys and values have one place each beside three parts of queries.
// Measured: 8 x 100 queries over 1444 keys, 8 heads of 32, 25 us (28 with a mask for each query); 4 x 2000 over 5776, 8 heads of 64, 652 us (145 TFLOP/s of f32 products; 32 on the CUDA cores).
// Few rows: the keys are split over the CTAs of a cluster, which join their sums through distributed shared memory.
#include <atomic>

#include "attention.cuh"

namespace dnb {

size_t tmem_smem(size_t bytes, int cols);
int conv_tc_max_smem();

namespace {

constexpr int KEYS = 64, SOFT = 8, CONVERT = 8, MMA_WARP = SOFT + CONVERT, THREADS = 640;
// Registers: 640 threads start with 96 each; 256 * 144 + 384 * 64 = 640 * 96.
constexpr int SOFT_REGS = 144, OTHER_REGS = 64;
constexpr int PASSES = 2;
constexpr uint32_t Q_BOX = 128 * 128, KV_BOX = KEYS * 128;   // 64 channels of a part: of the queries, of a tile's keys or values

struct alignas(16) F32TcShared {
    uint64_t q_full, k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], s_read[2], p_full[2], o_full, o_read, met[4];
    uint32_t tmem_base;
    int abort_flag;
    float halves[2][2][128];
};

struct F32TcArgs {
    AttnArgs a;
    int q_tokens, q_tiles, splits;
    float scale_log2;
};

template <int DP, bool MASK> struct F32TcCfg {
    static constexpr int BOXES = DP / 64, STAGES = DP == 64 ? 2 : 1, PITCH = DP + 4;
    static constexpr uint32_t Q_PART = BOXES * Q_BOX, KV_PART = BOXES * KV_BOX;
    static constexpr uint32_t K_AT = 3 * Q_PART, V_AT = K_AT + STAGES * 3 * KV_PART, WORK = V_AT + STAGES * 3 * KV_PART;
    static constexpr uint32_t MASKS_AT = WORK + sizeof(F32TcShared), BYTES = MASKS_AT + (MASK ? SOFT * MaskRows<32>::BYTES : 0);
    static constexpr uint32_t S_COL = 0, P_COL = 128, O_COL = 320;       // two of 64, two of 3 * 32, one of DP
    static_assert(130 * PITCH * 4 <= (int)WORK && BYTES <= 232448, "fits an SM");
};

// Eight channels of row r, channels 8c .., in three parts to their swizzled places.
__device__ __forceinline__ void store_parts(uint8_t *base, uint32_t box, uint32_t part, int r, int c, const float4 &x, const float4 &y)
{
    uint4 hi, mid, lo;
    split2(x.x, x.y, hi.x, mid.x, lo.x);
    split2(x.z, x.w, hi.y, mid.y, lo.y);
    split2(y.x, y.y, hi.z, mid.z, lo.z);
    split2(y.z, y.w, hi.w, mid.w, lo.w);
    uint8_t *to = base + (c >> 3) * box + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    *reinterpret_cast<uint4 *>(to) = hi;
    *reinterpret_cast<uint4 *>(to + part) = mid;
    *reinterpret_cast<uint4 *>(to + 2 * part) = lo;
}

__device__ __forceinline__ uint64_t desc_values64(uint32_t addr)        // rows of 64 channels, a key each: blocks of 64 channels a box apart, eight keys 1024 bytes
{
    uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(KV_BOX >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void tmem_ld_wait16(uint32_t *r)             // the values pass through the wait
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}

template <int DP, bool MASK>
__global__ void __launch_bounds__(THREADS, 1)
attention_f32_tc_kernel(const __grid_constant__ F32TcArgs t)
{
    using C = F32TcCfg<DP, MASK>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const AttnArgs &a = t.a;
    const uint32_t smem = smem_u32(smem_raw);
    if (smem & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, AT_SMEM_BASE);
        return;
    }
    F32TcShared *sh = reinterpret_cast<F32TcShared *>(smem_raw + C::WORK);
    volatile int *abort_flag = &sh->abort_flag;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = (int)(blockIdx.x % (unsigned)t.splits), job = (int)(blockIdx.x / (unsigned)t.splits);
    const int q_tile = job % t.q_tiles, kv_head = job / t.q_tiles % a.kv_heads, image = job / t.q_tiles / a.kv_heads;
    const int token0 = q_tile * t.q_tokens, rows_here = min(t.q_tokens, a.lq - token0) * a.group;

    if (tid == 0) {
        mbar_init(smem_u32(&sh->q_full), 16);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh->k_full[i]), CONVERT / 2);
            mbar_init(smem_u32(&sh->k_free[i]), 1);
            mbar_init(smem_u32(&sh->v_full[i]), CONVERT / 2);
            mbar_init(smem_u32(&sh->v_free[i]), 1);
            mbar_init(smem_u32(&sh->s_full[i]), 1);
            mbar_init(smem_u32(&sh->s_read[i]), SOFT);
            mbar_init(smem_u32(&sh->p_full[i]), SOFT);
        }
        mbar_init(smem_u32(&sh->o_full), 1);
        mbar_init(smem_u32(&sh->o_read), SOFT);
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&sh->met[i]), 2);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_dependency_wait();
    launch_dependents_if_small();
    const uint32_t tmem = sh->tmem_base;

    int keys = a.lk, first, tiles;
    if (a.lengths) keys = min(max(a.lengths[image], 0), a.lk);
    share_of_keys(keys, KEYS, rank, t.splits, first, tiles);
    const int steps = (a.d + 15) >> 4, chunks = 2 * steps;              // of 16 and of 8 channels

    auto finish = [&]() {
        if (*abort_flag) {                                              // products in flight end before their memory goes
            const long long begin = clock64();
            while (clock64() - begin < 4000000LL) { }
        }
        __syncthreads();
    };
    auto cluster_done = [&]() {
        __syncwarp();
        cluster_sync_all();
    };

    if (warp < MMA_WARP && tiles > 0) {
        for (int i = tid; i < 128 * chunks; i += MMA_WARP * 32) {
            const int r = i / chunks, c = i - r * chunks;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (r < rows_here && 8 * c < a.d) {
                const float4 *src = reinterpret_cast<const float4 *>((const float *)a.q + ((size_t)image * a.lq + token0 + r / a.group) * a.qp + (kv_head * a.group + r % a.group) * a.d + 8 * c);
                x = src[0];
                y = src[1];
            }
            store_parts(smem_raw, Q_BOX, C::Q_PART, r, c, x, y);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->q_full));
    }

    if (warp >= SOFT) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp < MMA_WARP) {
            // ------------------------------------------------------------ keys and values into parts
            const bool is_v = warp >= SOFT + CONVERT / 2;
            const int wt = tid & (CONVERT / 2 * 32 - 1);                // this thread among those of its operand
            const uint8_t *mask = a.mask && a.mask_query == 0 ? a.mask + (long long)image * a.mask_image : nullptr;
            const int pitch = is_v ? a.vp : a.kp;
            const float *src = (const float *)(is_v ? a.v : a.k) + (size_t)(a.kn == 1 ? 0 : image) * a.lk * pitch + kv_head * a.d;
            uint64_t *full = is_v ? sh->v_full : sh->k_full, *free_ = is_v ? sh->v_free : sh->k_free;
            // A pass: 2^turn lanes a row, eight channels each, a box's channels; PASSES of them are on their way while as many are split.
            const int turn = a.d > 32 ? 3 : a.d > 16 ? 2 : 1, c0 = wt & ((1 << turn) - 1), row0 = wt >> turn, pass_rows = CONVERT / 2 * 32 >> turn;
            const int per_box = (KEYS + PASSES * pass_rows - 1) / (PASSES * pass_rows), per_tile = per_box * ((a.d + 63) >> 6);
            struct Batch {
                float4 x[PASSES], y[PASSES];
            };
            auto load = [&](Batch &b, int j, int at) {
                const int c = (at >= per_box ? 8 : 0) + c0, base = (at >= per_box ? at - per_box : at) * PASSES * pass_rows + row0;
#pragma unroll
                for (int k = 0; k < PASSES; ++k) {
                    const int r = base + k * pass_rows, key = (first + j) * KEYS + r;
                    b.x[k] = b.y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    // zeros where there is no key, or none that any query sees
                    if (r < KEYS && key < keys && 8 * c < a.d && !(mask && !mask[key])) {
                        const float4 *p = reinterpret_cast<const float4 *>(src + (size_t)key * pitch + 8 * c);
                        b.x[k] = __ldg(p);
                        b.y[k] = __ldg(p + 1);
                    }
                }
            };
            int stage = 0;
            uint32_t phase = 0;
            Batch next;
            if (tiles > 0) load(next, 0, 0);
            for (int j = 0; j < tiles; ++j) {
                uint8_t *to = smem_raw + (is_v ? C::V_AT : C::K_AT) + stage * 3 * C::KV_PART;
#pragma unroll 1
                for (int at = 0; at < per_tile; ++at) {
                    const Batch b = next;
                    const bool last = at + 1 == per_tile;
                    if (!last || j + 1 < tiles) load(next, last ? j + 1 : j, last ? 0 : at + 1);
                    if (at == 0) mbar_wait_tight(smem_u32(&free_[stage]), phase ^ 1, abort_flag, a.status, AT_SLOT, a.polls);
                    const int c = (at >= per_box ? 8 : 0) + c0, base = (at >= per_box ? at - per_box : at) * PASSES * pass_rows + row0;
#pragma unroll
                    for (int k = 0; k < PASSES; ++k)
                        if (base + k * pass_rows < KEYS && c < chunks) store_parts(to, KV_BOX, C::KV_PART, base + k * pass_rows, c, b.x[k], b.y[k]);
                }
                fence_async_smem();
                __syncwarp();
                if (gave_up(abort_flag)) break;
                if (lane == 0 && !(a.debug & 32 && is_v)) mbar_arrive(smem_u32(&full[stage]));
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
        } else if (warp == MMA_WARP && tiles > 0) {
            // ------------------------------------------------------------ products
            const uint32_t idesc_qk = mma_idesc<MMA_BF16>(128, KEYS), idesc_pv = mma_idesc<MMA_BF16>(128, (uint32_t)(steps * 16)) | 1u << 16;   // bit 16: B's rows are contiguous along N
            const uint64_t dq = make_smem_desc(smem, 128), dk = make_smem_desc(smem + C::K_AT, 128), dv = desc_values64(smem + C::V_AT);
            auto wait = [&](uint64_t &bar, uint32_t parity, int code) { return mbar_wait_known(smem_u32(&bar), parity, abort_flag, a.status, code, a.polls); };
            int ks = 0, vs = 0;                                         // slots
            uint32_t kp = 0, vp = 0;
            auto scores = [&](int j) {
                if (elect_one()) {
                    const uint64_t k = dk + ks * (3 * C::KV_PART >> 4);
                    const uint32_t d = tmem + C::S_COL + (j & 1) * KEYS;
                    uint32_t add = 0;
#pragma unroll 1
                    for (int p = 0; p < 6; ++p) {
                        // (low, high) (high, low) (middle, middle) (middle, high) (high, middle) (high, high)
                        const uint32_t pa = 0x001102u >> (4 * p) & 15u, pb = 0x010120u >> (4 * p) & 15u;
                        const uint64_t qa = dq + pa * (C::Q_PART >> 4), kb = k + pb * (C::KV_PART >> 4);
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i)
                            if (i < steps) {
                                umma<MMA_BF16>(d, qa + ((i >> 2) * (Q_BOX >> 4) + (i & 3) * 2), kb + ((i >> 2) * (KV_BOX >> 4) + (i & 3) * 2), idesc_qk, add);
                                add = 1;
                            }
                    }
                    umma_commit(smem_u32(&sh->s_full[j & 1]));
                    umma_commit(smem_u32(&sh->k_free[ks]));
                }
                if (++ks == C::STAGES) { ks = 0; kp ^= 1; }
            };
            bool ok = wait(sh->q_full, 0, AT_QUERIES) && wait(sh->k_full[0], 0, AT_KEYS);
            if (ok) scores(0);
            for (int j = 0; ok && j < tiles; ++j) {
                if (j + 1 < tiles) {
                    ok = wait(sh->k_full[ks], kp, AT_KEYS) && (j < 1 || wait(sh->s_read[(j + 1) & 1], (j - 1) >> 1 & 1, AT_SCORES));
                    if (!ok) break;
                    tc_fence_after();
                    scores(j + 1);
                }
                ok = wait(sh->v_full[vs], vp, AT_VALUES) && (j < 1 || wait(sh->o_read, (j - 1) & 1, AT_OUTPUT)) && wait(sh->p_full[j & 1], j >> 1 & 1, AT_WEIGHTS);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t v = dv + vs * (3 * C::KV_PART >> 4);
                    const uint32_t p_at = tmem + C::P_COL + (j & 1) * 96;
#pragma unroll 1
                    for (int p = 0; p < 6; ++p) {
                        const uint32_t pa = 0x001102u >> (4 * p) & 15u, pb = 0x010120u >> (4 * p) & 15u;
#pragma unroll
                        for (int i = 0; i < KEYS / 16; ++i)
                            umma_from_tmem<false>(tmem + C::O_COL, p_at + pa * 32 + 8 * i, v + pb * (C::KV_PART >> 4) + i * (2048 >> 4), idesc_pv, p > 0 || i > 0);
                    }
                    umma_commit(smem_u32(&sh->o_full));
                    umma_commit(smem_u32(&sh->v_free[vs]));
                }
                if (++vs == C::STAGES) { vs = 0; vp ^= 1; }
            }
        }
        __syncwarp();
        __syncthreads();                                                // as below, where the rows are joined
        if (t.splits > 1) {
            cluster_done();
            cluster_done();
        }
        finish();
        if (warp == MMA_WARP) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        }
        return;
    }
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFT_REGS));

    // -------------------------------------------------------------------- softmax: half a row a thread, of the keys and of the channels
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const bool valid = row < rows_here;
    const int token = token0 + row / a.group;
    const uint32_t met = smem_u32(&sh->met[warp & 3]);
    const uint8_t *mask = nullptr;
    const uint32_t mask_at = smem + C::MASKS_AT + warp * MaskRows<32>::BYTES;
    if (MASK) {
        mask = a.mask + (long long)image * a.mask_image + (long long)(valid ? token : a.lq - 1) * a.mask_query;
        if (tiles > 0) mask_fetch<32>(mask_at, mask, first * KEYS + half * 32, keys, lane);
    }
    float o[DP / 2] = {}, top = -INFINITY, sum = 0.f;
    // adds the tile before, which was weighed against the same maximum as o
    auto add_tile = [&](int j, float shrink) {
        mbar_wait_tight(smem_u32(&sh->o_full), j & 1, abort_flag, a.status, AT_OUTPUT, a.polls);
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < DP / 2; c += 16)
            if (half * (DP / 2) + c < a.d) {
                uint32_t x[16];
                tmem_ld16(tmem + C::O_COL + lanes + half * (DP / 2) + c, x);
                tmem_ld_wait16(x);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[c + e] = (o[c + e] + __uint_as_float(x[e])) * shrink;
            }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->o_read));
    };
    for (int j = 0; j < tiles; ++j) {
        const int key0 = (first + j) * KEYS + half * 32, left = keys - key0;
        uint32_t bits = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
        if (MASK) {
            mask_bits<32>(mask_at, mask, key0, lane, &bits);
            if (j + 1 < tiles) mask_fetch<32>(mask_at, mask, key0 + KEYS, keys, lane);
        }
        mbar_wait_tight(smem_u32(&sh->s_full[j & 1]), j >> 1 & 1, abort_flag, a.status, AT_SCORES, a.polls);
        tc_fence_after();
        uint32_t v[32];
        const uint32_t s_at = tmem + C::S_COL + (j & 1) * KEYS + lanes + half * 32;
        tmem_ld16(s_at, *reinterpret_cast<uint32_t(*)[16]>(v));
        tmem_ld16(s_at + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
        tmem_ld_wait16(v);
        tmem_ld_wait16(v + 16);
        float grown = top;
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            float x = __uint_as_float(v[e]) * t.scale_log2, y = __uint_as_float(v[e + 1]) * t.scale_log2;
            if (!(bits >> e & 1)) x = -INFINITY;
            if (!(bits >> (e + 1) & 1)) y = -INFINITY;
            v[e] = __float_as_uint(x);
            v[e + 1] = __float_as_uint(y);
            grown = max3_nan(x, y, grown);                              // a NaN stays
        }
        sh->halves[j & 1][half][row] = grown;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(met);
            mbar_arrive(smem_u32(&sh->s_read[j & 1]));
        }
        mbar_wait_tight(met, j & 1, abort_flag, a.status, AT_SCORES, a.polls);
        grown = max3_nan(grown, sh->halves[j & 1][half ^ 1][row], grown);
        const float shrink = grown == top || top == -INFINITY ? (grown == top ? 1.f : 0.f) : ex2(top - grown);
        top = grown;
        const float base = top == -INFINITY ? 0.f : top;
        float now[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t hi[8], mid[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = ex2(__uint_as_float(v[c * 16 + 2 * e]) - base), y = ex2(__uint_as_float(v[c * 16 + 2 * e + 1]) - base);
                now[e & 1] += x + y;
                split2(x, y, hi[e], mid[e], lo[e]);
            }
            const uint32_t p_at = tmem + C::P_COL + (j & 1) * 96 + lanes + half * 16 + c * 8;
            tmem_st8(p_at, hi);
            tmem_st8(p_at + 32, mid);
            tmem_st8(p_at + 64, lo);
        }
        sum = sum * shrink + (now[0] + now[1]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh->p_full[j & 1]));
        if (j > 0) add_tile(j - 1, shrink);
    }
    if (tiles > 0) add_tile(tiles - 1, 1.f);
    sh->halves[0][half][row] = sum;                                     // (set 0 or 1 was compared before the last weights were waited for)
    __syncthreads();                                                    // every product has read its operands, too
    sum = sh->halves[0][0][row] + sh->halves[0][1][row];

    float *rows = reinterpret_cast<float *>(smem_raw), *tops = rows + 128 * C::PITCH, *sums = tops + 128;
    auto out = [&](int r) -> float * {
        return r >= rows_here ? nullptr : (float *)a.y + ((size_t)image * a.lq + token0 + r / a.group) * a.yp + (kv_head * a.group + r % a.group) * a.d;
    };
    if (t.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        float *y = out(row);
        if (y)
#pragma unroll
            for (int c = 0; c < DP / 2; c += 4)
                if (half * (DP / 2) + c < a.d) *reinterpret_cast<float4 *>(y + half * (DP / 2) + c) = make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
    } else {
        if (half == 0) {
            tops[row] = top;
            sums[row] = sum;
        }
#pragma unroll
        for (int c = 0; c < DP / 2; c += 4)
            *reinterpret_cast<float4 *>(rows + row * C::PITCH + half * (DP / 2) + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        cluster_done();
        if (!*abort_flag) join_rows<float>(smem_u32(rows), C::PITCH, smem_u32(tops), smem_u32(sums), min(rows_here, 128), a.d, rank, t.splits, tid, SOFT * 32, out);
        cluster_done();                                                 // a peer's rows are read until here
    }
    finish();
}

typedef void (*F32TcKernel)(F32TcArgs);

}  // namespace

bool attention_f32_tc_covers(const AttnArgs &a, int dtype)
{
    return dtype == DNB_F32 && a.d <= 128 && a.group <= 128 && (long long)a.n * a.kv_heads * ((a.lq + 127) / 128) * 128 < 1LL << 28;
}

int launch_attention_f32_tc(const AttnArgs &a, cudaStream_t stream)
{
    F32TcArgs t;
    t.a = a;
    t.q_tokens = 128 / a.group;
    t.q_tiles = (a.lq + t.q_tokens - 1) / t.q_tokens;
    t.scale_log2 = a.scale * 1.4426950408889634f;
    const int which = (a.d > 64 ? 2 : 0) + (a.mask ? 1 : 0);
    const F32TcKernel kern = which == 0 ? attention_f32_tc_kernel<64, false> : which == 1 ? attention_f32_tc_kernel<64, true>
                             : which == 2 ? attention_f32_tc_kernel<128, false> : attention_f32_tc_kernel<128, true>;
    static std::atomic<bool> done[64][4];
    int dev = 0;
    DNB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) DNB_FAIL(DNB_ECUDA, "attention: device %d", dev);
    if (!done[dev][which].load(std::memory_order_acquire)) {
        DNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, conv_tc_max_smem()));
        done[dev][which].store(true, std::memory_order_release);
    }
    const long long jobs = (long long)a.n * a.kv_heads * t.q_tiles;
    const int key_tiles = (a.lk + KEYS - 1) / KEYS;
    const size_t bytes = tmem_smem(a.mask ? (a.d > 64 ? F32TcCfg<128, true>::BYTES : F32TcCfg<64, true>::BYTES) : a.d > 64 ? F32TcCfg<128, false>::BYTES : F32TcCfg<64, false>::BYTES, 512);
    // Heads of 64, us over 1 / 2 / 4 / 8 CTAs a job: 8 jobs of 6 tiles 17.6 / 14.3 / 12.6 / 15.1, 32 jobs of 23 49.0 / 31.5 / 21.6 / 51.6, 200 jobs of 91
    // 360 / 295 / 380.  A tile's time is 1.9 us (4.6 of heads of 128); one pair of constants serves both.  The images' own lengths are on the device and do not
    // count: 256 jobs of up to 91 tiles 283 / 265 / 316, as chosen 283.
    int room[4];
    DNB_TRY(cluster_room((const void *)kern, 4 + which, THREADS, bytes, room));
    t.splits = split_keys(jobs, key_tiles, room, 3.0, 0.5);
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = pdl_enabled() && jobs * t.splits <= EARLY_BLOCKS ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = (unsigned)t.splits; attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(jobs * t.splits));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    DNB_CUDA(cudaLaunchKernelEx(&cfg, kern, t));
    DNB_LAUNCH_CHECK("attention");
    return DNB_OK;
}

}  // namespace dnb
