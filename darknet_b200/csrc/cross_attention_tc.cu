// Cross attention of bf16 tensors on the 5th-generation tensor cores.
//
// A CTA holds two tiles of 128 query rows (a row: one query token of one head; the heads that share keys lie side by side, so that their keys
// are loaded once) and walks over the keys in tiles of 128:
//   S = Q K^T   tcgen05.mma, both operands in shared memory by TMA, S in TMEM (fp32)
//   P = exp2(S * scale * log2 e - m)   eight warps a tile, half a row a thread, out of TMEM and back into it as bf16
//   O += P V    tcgen05.mma, P from TMEM, V from shared memory as it lies (channels innermost: a transposed operand), O in TMEM (fp32)
// While one tile's warps take exponentials, the tensor cores multiply the other tile's: the two are never both idle.
// Measured: 8 x 5776 queries over 5776 keys, 8 heads of 128 916 us on a cool GPU (1190 TFLOP/s, tensor pipe and exponentials 58 % each) and 1055 to 1073 us
// (1020 TFLOP/s) in a run of seconds, under the power cap; of 64 710 us (770 TFLOP/s): there
// the softmax's chain bounds it (exponentials for nothing would save 4 %; a share of them as polynomials on the FMA pipe costs 4 to 10 %).
//
// The running maximum m moves only when a row's largest score has outgrown it by more than 2^8 (every weight is then at most 256 times what
// the largest should be, far inside bf16's and fp32's range); until then O needs no correction.  The sum of the weights is kept in fp32 of the
// unrounded weights; a weight is rounded to bf16 (half a step: 2^-8 of itself) as the operand of the second product, and nothing else is rounded
// before the output.
//
// Few rows: the keys of one pair of tiles are split over the CTAs of a cluster, which join their sums through distributed shared memory: no
// workspace, one launch, the same order of additions every time.
#include <atomic>

#include "attention.cuh"

namespace dnb {

int encode_tensor_map(CUtensorMap *map, int elem_kind, int rank, void *base, const uint64_t *dims, const uint64_t *strides_bytes, const uint32_t *box, int swizzle_bytes);
size_t tmem_smem(size_t bytes, int cols);
int conv_tc_max_smem();

namespace {

constexpr int SOFT_WARPS = 16, LOAD_WARP = 16, MMA_WARP = 17, THREADS = 20 * 32;
// Registers: 640 threads start with 96 each; the four warps that load and multiply give 32 back, the sixteen others take 8 more: 512 * 104 + 128 * 64 = 640 * 96.
constexpr int SOFT_REGS = 104, OTHER_REGS = 64;
constexpr int MAX_STAGES = 12;
constexpr uint32_t BOX_BYTES = 128 * 128;         // 64 channels of 128 rows
constexpr float MOVE = 8.f;                       // how far (log2) scores may outgrow the running maximum

struct alignas(16) Shared {
    uint64_t q_full, full[MAX_STAGES], empty[MAX_STAGES], s_full[2], s_read[2], p_full[2], o_full[2], met[8];
    uint32_t tmem_base;
    int abort_flag;
    float halves[][2][256];                       // the largest scores of the rows' halves, and their sums at the end
};

struct alignas(64) TcAttnArgs {
    CUtensorMap tmq, tmk, tmv;
    AttnArgs a;
    int q_tokens;          // query tokens of a tile
    int q_tiles;           // pairs of tiles an image and key head
    int splits;            // CTAs of a cluster
    float scale_log2;      // |scale| * log2 e
    int negate;            // scale < 0: the products with -Q
};

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t *r)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
          "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// Waits for the loads so far; the values pass through it, so that nothing that uses them is moved in front of it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t *r)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
// V as it lies in shared memory: rows of 64 channels (128 bytes, swizzled), a key each: N is contiguous.  Blocks of 64 channels are a box
// apart, groups of eight keys 1024 bytes.
__device__ __forceinline__ uint64_t desc_values(uint32_t addr)
{
    uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(BOX_BYTES >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// DP: channels of a head as they lie in shared memory, 64 or 128 (TMA fills what the head does not have with zeros).
template <int DP, bool MASK> struct Cfg {
    static constexpr int BOXES = DP / 64;
    static constexpr uint32_t TILE_BYTES = BOXES * BOX_BYTES;
    static constexpr int STAGES = DP == 128 ? (MASK ? 3 : 5) : MASK ? 9 : 11;
    static constexpr uint32_t WORK = 2 * TILE_BYTES + STAGES * TILE_BYTES;
    static constexpr int PITCH = DP + 4;          // of a row of sums, for the join
    // TMEM: the scores of both tiles, their outputs and, where there is room, weights of their own.  Then the next tile's scores are made while the
    // weights of this one are; heads of more than 64 channels have the weights in the scores' place, and the next scores wait for their product.
    static constexpr bool OWN_P = DP == 64;
    static constexpr uint32_t O_AT = 256, P_AT = OWN_P ? 256 + 2 * DP : 0, P_STEP = OWN_P ? 64 : 128;
    // The halves' largest scores: one set for each of two tiles of keys where the next scores may be there before this tile's have been compared.
    static constexpr int SETS = OWN_P ? 2 : 1;
    static constexpr uint32_t MASKS_AT = WORK + sizeof(Shared) + SETS * 2048, BYTES = MASKS_AT + (MASK ? SOFT_WARPS * MaskRows<64>::BYTES : 0);
    static_assert(258 * PITCH * 4 + 2048 <= WORK && STAGES <= MAX_STAGES, "the rows' sums fit where the operands were");
    static_assert(BYTES <= 232448, "fits an SM");
};

template <int DP, bool MASK>
__global__ void __launch_bounds__(THREADS, 1)
attention_tc_kernel(const __grid_constant__ TcAttnArgs t)
{
    using C = Cfg<DP, MASK>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const AttnArgs &a = t.a;
    const uint32_t smem = smem_u32(smem_raw);
    if (smem & 1023u) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, AT_SMEM_BASE);
        return;
    }
    Shared *sh = reinterpret_cast<Shared *>(smem_raw + C::WORK);
    volatile int *abort_flag = &sh->abort_flag;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t q_smem = smem, ring = smem + 2 * C::TILE_BYTES;

    const int rank = (int)(blockIdx.x % (unsigned)t.splits), job = (int)(blockIdx.x / (unsigned)t.splits);
    const int q_tile = job % t.q_tiles, kv_head = job / t.q_tiles % a.kv_heads, image = job / t.q_tiles / a.kv_heads;
    const int token0 = q_tile * 2 * t.q_tokens;
    const int sides = token0 + t.q_tokens < a.lq ? 2 : 1;

    if (tid == 0) {
        mbar_init(smem_u32(&sh->q_full), 1);
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(smem_u32(&sh->full[i]), 1);
            mbar_init(smem_u32(&sh->empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh->s_full[i]), 1);
            mbar_init(smem_u32(&sh->s_read[i]), 8);
            mbar_init(smem_u32(&sh->p_full[i]), 8);
            mbar_init(smem_u32(&sh->o_full[i]), 1);
        }
        for (int i = 0; i < 8; ++i) mbar_init(smem_u32(&sh->met[i]), 2);
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
    auto s_cols = [&](int s) { return tmem + 128 * s; };
    auto o_cols = [&](int s) { return tmem + C::O_AT + DP * s; };
    auto p_cols = [&](int s) { return tmem + C::P_AT + C::P_STEP * s; };

    int keys = a.lk;
    if (a.lengths) keys = min(max(a.lengths[image], 0), a.lk);
    int t0, tiles;
    share_of_keys(keys, 128, rank, t.splits, t0, tiles);

    auto cluster_done = [&]() {
        __syncwarp();
        cluster_sync_all();
    };
    auto finish = [&]() {
        if (*abort_flag) {                                              // loads and products in flight end before their memory goes
            const long long begin = clock64();
            while (clock64() - begin < 4000000LL) { }
        }
        __syncthreads();
    };
    if (warp >= SOFT_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == LOAD_WARP) {
        // ---------------------------------------------------------------- loads
        if (tiles > 0) {
            const int kv_image = a.kn == 1 ? 0 : image;
            const uint32_t q_bytes = (uint32_t)(a.group * t.q_tokens) * 128u;
            const uint32_t qbar = smem_u32(&sh->q_full);
            if (elect_one()) {
                mbar_expect_tx(qbar, q_bytes * C::BOXES * sides);
                for (int s = 0; s < sides; ++s)
                    for (int b = 0; b < C::BOXES; ++b)
                        tma_load_4d(q_smem + s * C::TILE_BYTES + b * BOX_BYTES, &t.tmq, qbar, b * 64, kv_head * a.group, token0 + s * t.q_tokens, image);
            }
            int stage = 0;
            uint32_t phase = 0;
            for (int i = 0; i < 2 * tiles; ++i) {
                const uint32_t full = smem_u32(&sh->full[stage]);
                if (!mbar_wait_known(smem_u32(&sh->empty[stage]), phase ^ 1, abort_flag, a.status, AT_SLOT, a.polls) || gave_up(abort_flag)) break;
                if (elect_one() && !(a.debug & 32 && i == 1)) {
                    mbar_expect_tx(full, C::TILE_BYTES);
                    for (int b = 0; b < C::BOXES; ++b)
                        tma_load_4d(ring + stage * C::TILE_BYTES + b * BOX_BYTES, i & 1 ? &t.tmv : &t.tmk, full, b * 64, kv_head, (t0 + i / 2) * 128, kv_image);
                }
                if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == MMA_WARP) {
        // ---------------------------------------------------------------- products
        bool ok = tiles > 0 && mbar_wait_known(smem_u32(&sh->q_full), 0, abort_flag, a.status, AT_QUERIES, a.polls);
        const int qk_steps = (a.d + 15) >> 4;
        const uint32_t idesc_qk = mma_idesc<MMA_BF16>(128, 128) | (t.negate ? 1u << 13 : 0u);                     // bit 13: A, negated
        const uint32_t idesc_pv = mma_idesc<MMA_BF16>(128, (uint32_t)(qk_steps * 16)) | 1u << 16;                 // bit 16: B's rows are contiguous along N
        const uint64_t dq = make_smem_desc(q_smem, 128), dk = make_smem_desc(ring, 128), dv = desc_values(ring);
        constexpr uint64_t SLOT = C::TILE_BYTES >> 4;
        // Descriptors are a base and constants, products are unrolled: with their addresses made one by one the issue of a product took 55 clocks, as long
        // as the product.
        auto scores = [&](int s, int slot) {
            if (elect_one()) {
                const uint64_t q = dq + s * SLOT, k = dk + slot * SLOT;
                if (qk_steps == DP / 16) {
                    umma<MMA_BF16>(s_cols(s), q, k, idesc_qk, 0u);
#pragma unroll
                    for (int i = 1; i < DP / 16; ++i) {
                        const uint64_t off = ((i >> 2) * BOX_BYTES + (i & 3) * 32) >> 4;
                        umma<MMA_BF16>(s_cols(s), q + off, k + off, idesc_qk, 1u);
                    }
                } else {
                    for (int i = 0; i < qk_steps; ++i) {
                        const uint64_t off = ((i >> 2) * BOX_BYTES + (i & 3) * 32) >> 4;
                        umma<MMA_BF16>(s_cols(s), q + off, k + off, idesc_qk, i > 0);
                    }
                }
                umma_commit(smem_u32(&sh->s_full[s]));
            }
        };
        auto output = [&](int s, int slot, uint32_t add, bool done) {
            if (elect_one()) {
                const uint64_t v = dv + slot * SLOT;
                umma_from_tmem<false>(o_cols(s), p_cols(s), v, idesc_pv, add);
#pragma unroll
                for (int i = 1; i < 8; ++i) umma_from_tmem<true>(o_cols(s), p_cols(s) + 8 * i, v + i * (2048 >> 4), idesc_pv, 1u);
                if (done) umma_commit(smem_u32(&sh->o_full[s]));
            }
        };
        auto release = [&](int slot) {
            if (elect_one()) umma_commit(smem_u32(&sh->empty[slot]));
        };
        auto landed = [&](int slot, uint32_t phase, int code) { return mbar_wait_known(smem_u32(&sh->full[slot]), phase, abort_flag, a.status, code, a.polls); };
        // slot 2j of the ring is K's tile j, slot 2j + 1 V's
        int stage = 0;
        uint32_t phase = 0;
        auto next = [&]() { if (++stage == C::STAGES) { stage = 0; phase ^= 1; } };
        ok = ok && landed(0, 0, AT_KEYS);
        if (ok) {
            scores(0, 0);
            if (sides == 2) {
                // The tiles take turns: one looks for its largest scores while the other's exponentials go through.  Where each has its scores in time they
                // stay as they start, and started together they keep both pipes waiting in turn (8 x 1444 x 5776 tokens, 8 heads of 64: 269 us, and 211 so).
                if (C::OWN_P) ok = mbar_wait_known(smem_u32(&sh->s_read[0]), 0, abort_flag, a.status, AT_SCORES, a.polls);
                if (ok) scores(1, 0);
            }
            release(0);
            next();
        }
        for (int j = 0; ok && j < tiles; ++j) {
            const int v_slot = stage;
            const uint32_t v_phase = phase;
            next();
            const int k_slot = stage;
            const uint32_t k_phase = phase;
            const bool more = j + 1 < tiles;
            // operands first, while the weights are being made
            ok = landed(v_slot, v_phase, AT_VALUES);
            if (more) {
                next();
                ok = ok && landed(k_slot, k_phase, AT_KEYS);
            }
            if (!ok) break;
            if constexpr (C::OWN_P) {
                if (more) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        if (s < sides && ok) {
                            ok = mbar_wait_known(smem_u32(&sh->s_read[s]), j & 1, abort_flag, a.status, AT_SCORES, a.polls);
                            tc_fence_after();
                            if (ok) scores(s, k_slot);
                        }
                    if (!ok) break;
                    release(k_slot);
                }
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (s < sides && ok) {
                        ok = mbar_wait_known(smem_u32(&sh->p_full[s]), j & 1, abort_flag, a.status, AT_WEIGHTS, a.polls);
                        tc_fence_after();
                        if (ok) output(s, v_slot, j > 0, true);
                    }
                if (!ok) break;
                release(v_slot);
            } else {
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (s < sides && ok) {
                        ok = mbar_wait_known(smem_u32(&sh->p_full[s]), j & 1, abort_flag, a.status, AT_WEIGHTS, a.polls);
                        tc_fence_after();
                        if (ok) {
                            output(s, v_slot, j > 0, !more);
                            if (more) scores(s, k_slot);
                        }
                    }
                if (!ok) break;
                release(v_slot);
                if (more) release(k_slot);
            }
        }
    }
    __syncwarp();
    __syncthreads();                                                    // as below, where the rows are joined
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

    // ---------------------------------------------------------------- softmax: half a row a thread
    const int s = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const bool mine = warp < 8 * sides;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;                  // this warp's lanes of TMEM
    const int r_token = token0 + s * t.q_tokens + row / a.group;
    const bool valid = mine && row < t.q_tokens * a.group && r_token < a.lq;
    float top = -INFINITY, sum = 0.f;
    if (mine) {
        const float scale = t.scale_log2;
        const uint32_t met = smem_u32(&sh->met[s * 4 + (warp & 3)]);    // this warp and the one with the rows' other half
        const uint8_t *mask = nullptr;
        const uint32_t mask_at = smem + C::MASKS_AT + warp * MaskRows<64>::BYTES;
        if (MASK) {
            mask = a.mask + (long long)image * a.mask_image + (valid ? r_token : a.lq - 1) * a.mask_query;
            if (tiles > 0) mask_fetch<64>(mask_at, mask, t0 * 128 + half * 64, keys, lane);
        }
        int stage = 1;
        uint32_t phase = 0;                                             // of V's slots
        for (int j = 0; j < tiles; ++j) {
            const int key0 = (t0 + j) * 128, left = keys - key0, col0 = half * 64;
            uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
            uint8_t seen = 1;                                           // with one mask for all queries: key `row` of the tile
            if (MASK) {
                mask_bits<64>(mask_at, mask, key0 + col0, lane, bits);
                if (j + 1 < tiles) mask_fetch<64>(mask_at, mask, key0 + 128 + col0, keys, lane);
                if (a.mask_query == 0 && row < left) seen = mask[key0 + row];
            } else if (left < 128) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const int n = left - col0 - 32 * w;
                    bits[w] = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
                }
            }
            mbar_wait_tight(smem_u32(&sh->s_full[s]), j & 1, abort_flag, a.status, AT_SCORES, a.polls);
            tc_fence_after();
            uint32_t v[64];
            float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_ld32(s_cols(s) + lanes + col0, v);
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                tmem_ld_wait32(v + c);
                if (c == 0) tmem_ld32(s_cols(s) + lanes + col0 + 32, v + 32);             // travels while the first ones' largest is looked for
                if (MASK || left < 128) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(bits[c >> 5] >> e & 1)) v[c + e] = 0xff800000u;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 2) most[e / 2 & 3] = max3_nan(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1]), most[e / 2 & 3]);
            }
            float grown = max3_nan(max3_nan(most[0], most[1], most[2]), most[3], top);    // a NaN stays
            // The halves of a row meet.  After it both have read their scores: the weights may take their place.
            sh->halves[j & (C::SETS - 1)][half][s * 128 + row] = grown;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(met);
                if (C::OWN_P) mbar_arrive(smem_u32(&sh->s_read[s]));
            }
            mbar_wait_tight(met, j & 1, abort_flag, a.status, AT_SCORES, a.polls);
            tc_fence_after();
            grown = max3_nan(grown, sh->halves[j & (C::SETS - 1)][half ^ 1][s * 128 + row], grown);
            // The tile before has to be out of O (its corrections) and, with a place of its own, of P.
            if (C::OWN_P && j > 0) {
                mbar_wait_tight(smem_u32(&sh->o_full[s]), (j - 1) & 1, abort_flag, a.status, AT_OUTPUT, a.polls);
                tc_fence_after();
            }
            // A row that no query fills has no say: its queries are what an earlier kernel left in shared memory, where the heads of a tile are no 128.
            if (__any_sync(0xffffffffu, valid && !((grown - top) * scale <= MOVE) && grown != -INFINITY)) {
                const float shrink = grown == top ? 1.f : ex2((top - grown) * scale);
                if (j > 0) {
                    // each half its half of the channels (without a place of its own for P every product of the tile before has retired: the
                    // scores' barrier came after them)
#pragma unroll 1
                    for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_cols(s) + lanes + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                        tmem_st16(o_cols(s) + lanes + c, o);
                    }
                }
                sum *= shrink;
                top = grown;
            }
            const float base = top == -INFINITY ? 0.f : top * scale;
            const uint64_t scale2 = pack2(scale, scale), base2 = pack2(-base, -base);
            uint64_t sums[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x, y;
                    unpack2(fma2(pack2(__uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1])), scale2, base2), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    sums[e & 1] = add2(sums[e & 1], pack2(x, y));
                    p[e] = pack_bf16(x, y);
                }
                tmem_st16(p_cols(s) + lanes + (col0 + c) / 2, p);
            }
            float x0, x1;
            unpack2(add2(sums[0], sums[1]), x0, x1);
            sum += x0 + x1;
            // Values that no weight reaches may be anything, and zero times infinity is no number: zeros in their place.  (Both tiles write them.)
            if ((left < 128 && keys < a.lk) || (MASK && a.mask_query == 0)) {
                mbar_wait_tight(smem_u32(&sh->full[stage]), phase, abort_flag, a.status, AT_VALUES, a.polls);
                if (row >= left || (MASK && !seen)) {
                    const uint32_t at = 2 * C::TILE_BYTES + stage * C::TILE_BYTES + row * 128;
#pragma unroll
                    for (int b = half; b < C::BOXES; b += 2)
#pragma unroll
                        for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4 *>(smem_raw + at + b * BOX_BYTES + e * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            stage += 2;
            if (stage >= C::STAGES) { stage -= C::STAGES; phase ^= 1; }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->p_full[s]));
        }
        if (tiles > 0) {
            mbar_wait_tight(smem_u32(&sh->o_full[s]), C::OWN_P ? (tiles - 1) & 1 : 0, abort_flag, a.status, AT_OUTPUT, a.polls);
            tc_fence_after();
        }
        sh->halves[0][half][s * 128 + row] = sum;                       // the other half has compared its last: its weights were waited for
    }
    __syncthreads();                                                    // every product has read its operands, too
    if (mine) sum = sh->halves[0][0][s * 128 + row] + sh->halves[0][1][s * 128 + row];

    const bool wide = a.d % 16 == 0 && a.yp % 16 == 0 && (uintptr_t)a.y % 32 == 0;   // whole 32-byte sectors
    __nv_bfloat16 *y = (__nv_bfloat16 *)a.y + ((size_t)image * a.lq + r_token) * a.yp + (kv_head * a.group + row % a.group) * a.d;
    const int o0 = half * (DP / 2), o1 = min(o0 + DP / 2, a.d);         // this thread's channels
    if (t.splits == 1) {
        if (mine) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll 1
            for (int c = o0; c < o1; c += 16) {
                uint32_t o[16], p[8];
                if (tiles > 0) {
                    tmem_ld16(o_cols(s) + lanes + c, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    p[e] = tiles > 0 && sum != 0.f ? pack_bf16(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv) : 0u;
                if (valid) {
                    if (wide) st_global_32(y + c, p);
                    else {
                        *reinterpret_cast<uint4 *>(y + c) = make_uint4(p[0], p[1], p[2], p[3]);
                        if (c + 8 < a.d) *reinterpret_cast<uint4 *>(y + c + 8) = make_uint4(p[4], p[5], p[6], p[7]);
                    }
                }
            }
        }
    } else {
        float *rows = reinterpret_cast<float *>(smem_raw), *tops = rows + 256 * C::PITCH, *sums = tops + 256;
        if (mine) {
            if (half == 0) {
                tops[s * 128 + row] = top * t.scale_log2;
                sums[s * 128 + row] = sum;
            }
            if (tiles > 0) {
#pragma unroll 1
                for (int c = o0; c < o1; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(o_cols(s) + lanes + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<uint4 *>(rows + (s * 128 + row) * C::PITCH + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
        }
        cluster_done();
        if (!*abort_flag)
            join_rows<__nv_bfloat16>(smem_u32(rows), C::PITCH, smem_u32(tops), smem_u32(sums), 128 * sides, a.d, rank, t.splits, tid, SOFT_WARPS * 32, [&](int r) -> __nv_bfloat16 * {
                const int in_tile = r & 127, token = token0 + (r >> 7) * t.q_tokens + in_tile / a.group;
                if (in_tile >= t.q_tokens * a.group || token >= a.lq) return nullptr;
                return (__nv_bfloat16 *)a.y + ((size_t)image * a.lq + token) * a.yp + (kv_head * a.group + in_tile % a.group) * a.d;
            });
        cluster_done();                                                 // a peer's rows are read until here
    }
    finish();
}

typedef void (*Kernel)(TcAttnArgs);

int prepare(Kernel kern, int which)
{
    static std::atomic<bool> done[64][4];
    int dev = 0;
    DNB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) DNB_FAIL(DNB_ECUDA, "attention: device %d", dev);
    if (done[dev][which].load(std::memory_order_acquire)) return DNB_OK;
    DNB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, conv_tc_max_smem()));
    done[dev][which].store(true, std::memory_order_release);
    return DNB_OK;
}

}  // namespace

bool attention_tc_covers(const AttnArgs &a, int dtype)
{
    const long long jobs = (long long)a.n * a.kv_heads * ((a.lq + 127) / 128) * 128;
    return dtype == DNB_BF16 && a.d <= 128 && a.group <= 128 && jobs < 1LL << 28;
}

int launch_attention_tc(const AttnArgs &a, cudaStream_t stream)
{
    TcAttnArgs t;
    t.a = a;
    t.q_tokens = 128 / a.group;
    t.q_tiles = (a.lq + 2 * t.q_tokens - 1) / (2 * t.q_tokens);
    t.scale_log2 = (a.scale < 0.f ? -a.scale : a.scale) * 1.4426950408889634f;
    t.negate = a.scale < 0.f;
    auto map = [&](CUtensorMap *m, const void *data, int heads, int pitch, int tokens, int images, int box_heads, int box_tokens) {
        const uint64_t dims[4] = {(uint64_t)a.d, (uint64_t)heads, (uint64_t)tokens, (uint64_t)images};
        const uint64_t strides[3] = {(uint64_t)a.d * 2, (uint64_t)pitch * 2, (uint64_t)tokens * pitch * 2};
        const uint32_t box[4] = {64, (uint32_t)box_heads, (uint32_t)box_tokens, 1};
        return encode_tensor_map(m, 1, 4, const_cast<void *>(data), dims, strides, box, 128);
    };
    DNB_TRY(map(&t.tmq, a.q, a.heads, a.qp, a.lq, a.n, a.group, t.q_tokens));
    DNB_TRY(map(&t.tmk, a.k, a.kv_heads, a.kp, a.lk, a.kn, 1, 128));
    DNB_TRY(map(&t.tmv, a.v, a.kv_heads, a.vp, a.lk, a.kn, 1, 128));
    const long long jobs = (long long)a.n * a.kv_heads * t.q_tiles;
    const int key_tiles = (a.lk + 127) / 128;
    const int which = (a.d > 64 ? 2 : 0) + (a.mask ? 1 : 0);
    const Kernel kern = which == 0 ? attention_tc_kernel<64, false> : which == 1 ? attention_tc_kernel<64, true> : which == 2 ? attention_tc_kernel<128, false> : attention_tc_kernel<128, true>;
    DNB_TRY(prepare(kern, which));
    const size_t bytes = tmem_smem(a.mask ? (a.d > 64 ? Cfg<128, true>::BYTES : Cfg<64, true>::BYTES) : a.d > 64 ? Cfg<128, false>::BYTES : Cfg<64, false>::BYTES, 512);
    // Heads of 64, us over 1 / 2 / 4 / 8 CTAs a job: 8 jobs of 3 tiles 9.5 / 11.4 / 13.5, of 12 22.8 / 17.0 / 15.1 / 19.3, of 46 69.7 / 41.2 / 27.8 / 25.4;
    // 152 jobs of 46 144 / 128 / 145, 384 jobs of 46 216 / 249.  A tile's time is 1.4 us (1.8 of heads of 128); one pair of constants serves both.  The images' own
    // lengths are on the device and do not count: 128 jobs of up to 46 tiles 73.4 / 72.9 / 99.2, as chosen 73.4.
    int room[4];
    DNB_TRY(cluster_room((const void *)kern, which, THREADS, bytes, room));
    t.splits = a.mask ? split_keys(jobs, key_tiles, room, 2.5, 0.6) : split_keys(jobs, key_tiles, room, 4.0, 1.0);   // a masked tile takes 1.7 times as long
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
