// Attention of query tokens to an encoder's states (a feature map's pixels): plan, checks, choice of the kernel, and the kernel for every case.
//
//   s_ij = scale * q_i . k_j      o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)      over the keys j that query i may see, m_i their largest s
//
// A query that may see no key gets zeros.
#include <math.h>

#include <atomic>
#include <new>

#include "attention.h"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

namespace dnb {

constexpr float LOG2E = 1.4426950408889634f;

// One warp a query and head: 32 keys at a time, a key a lane for the scores, a few channels a lane for the sum of the values, the largest score and
// the sum of the weights as they go.  Right for every case; what is left to it are more than 128 heads a key head, more than a tile of the others holds.
// A lane's loads of its key, one channel after another, bound it: 8 tokens, 160 heads of 64 over one key head and 1444 keys, 829 us in bf16 and 946 in f32,
// where 128 heads take the tensor cores 10 and 19.
template <typename T>
__global__ void __launch_bounds__(128)
attention_simple_kernel(const __grid_constant__ AttnArgs a)
{
    __shared__ float rows[4][128];
    grid_dependency_wait();
    launch_dependents_if_small();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + warp, total = (long long)a.n * a.lq * a.heads;
    if (row >= total) return;
    const int head = (int)(row % a.heads), image = (int)(row / a.heads / a.lq);
    const long long token = row / a.heads;
    const T *q = (const T *)a.q + (size_t)token * a.qp + head * a.d;
    for (int i = lane; i < a.d; i += 32) rows[warp][i] = to_float<T>(q[i]);
    __syncwarp();
    const size_t first = (size_t)(a.kn == 1 ? 0 : image) * a.lk;
    const T *k = (const T *)a.k + first * a.kp + head / a.group * a.d, *v = (const T *)a.v + first * a.vp + head / a.group * a.d;
    int keys = a.lk;
    if (a.lengths) keys = min(max(a.lengths[image], 0), a.lk);
    const uint8_t *mask = a.mask ? a.mask + image * a.mask_image + (token - (long long)image * a.lq) * a.mask_query : nullptr;
    const float scale = a.scale * LOG2E;
    float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < keys; j0 += 32) {
        const int j = j0 + lane;
        const bool in = j < keys && (!mask || mask[j]);
        float s = -INFINITY;
        if (in) {
            const T *kr = k + (size_t)j * a.kp;
            float dot = 0.f;
            for (int i = 0; i < a.d; ++i) dot = fmaf(rows[warp][i], to_float<T>(kr[i]), dot);
            s = dot * scale;
        }
        float most = s;
#pragma unroll
        for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        const float next = fmaxf(top, most), base = next == -INFINITY ? 0.f : next;
        const float shrink = exp2f(top - base);
        float p = in ? exp2f(s - base) : 0.f;
        top = next;
        sum *= shrink;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= shrink;
        sum += p;
        const unsigned seen = __ballot_sync(0xffffffffu, in);
        for (int i = 0; i < 32; ++i) {
            const float w = __shfl_sync(0xffffffffu, p, i);
            if (!(seen >> i & 1)) continue;                     // what lies behind a mask is not read
            const T *vr = v + (size_t)(j0 + i) * a.vp;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 32 * c < a.d) o[c] = fmaf(w, to_float<T>(vr[lane + 32 * c]), o[c]);
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    T *y = (T *)a.y + (size_t)token * a.yp + head * a.d;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < a.d) y[lane + 32 * c] = from_float<T>(sum == 0.f ? 0.f : o[c] / sum);
}

int launch_attention_simple(const AttnArgs &a, int dtype, cudaStream_t s)
{
    const long long rows = (long long)a.n * a.lq * a.heads, blocks = (rows + 3) / 4;
    if (blocks >= 1LL << 31) DNB_FAIL(DNB_EUNSUPPORTED, "attention: %lld rows", rows);
    if (dtype == DNB_BF16) DNB_CUDA(launch_overlapped(attention_simple_kernel<__nv_bfloat16>, dim3((unsigned)blocks), 128, 0, s, a));
    else DNB_CUDA(launch_overlapped(attention_simple_kernel<float>, dim3((unsigned)blocks), 128, 0, s, a));
    DNB_LAUNCH_CHECK("attention");
    return DNB_OK;
}

int split_keys(long long jobs, int key_tiles, const int room[4], double start, double join)
{
    int best = 1;
    double least = 0.0;
    for (int i = 0, s = 1; i < 4 && (s == 1 || s <= key_tiles); ++i, s *= 2) {
        if (room[i] < s) continue;
        const double waves = (double)((jobs * s + room[i] - 1) / room[i]), cost = waves * ((key_tiles + s - 1) / s + start + (s > 1 ? join * s : 0.0));
        if (s == 1 || cost < least) {
            best = s;
            least = cost;
        }
    }
    return best;
}

int cluster_room(const void *kernel, int slot, int threads, size_t smem, int room[4])
{
    static std::atomic<int> known[64][8][4];
    int dev = 0;
    DNB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) DNB_FAIL(DNB_ECUDA, "attention: device %d", dev);
    for (int i = 0; i < 4; ++i) {
        room[i] = known[dev][slot][i].load(std::memory_order_relaxed);
        if (room[i]) continue;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 1u << i; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1u << i);
        cfg.blockDim = dim3((unsigned)threads);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        DNB_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
        room[i] = clusters > 0 ? clusters << i : i == 0 ? sm_count() : -1;
        known[dev][slot][i].store(room[i], std::memory_order_relaxed);
    }
    return DNB_OK;
}

// Whether a tensor reaches into a mask's bytes: `queries` rows of `keys` bytes an image, at the mask's strides.
static bool reaches_into_mask(const dnb_tensor *t, const dnb_attention_mask *m, int images, int queries, int keys)
{
    const __int128 image = images > 1 ? m->image_stride : 0, query = queries > 1 ? m->query_stride : 0, whole = (images - 1) * image + (queries - 1) * query + keys;
    const uintptr_t at = (uintptr_t)m->mask;
    if (!reaches_into(t, m->mask, whole > (__int128)(UINTPTR_MAX - at) ? (size_t)(UINTPTR_MAX - at) : (size_t)whole)) return false;
    // between the first and the last byte: the first row of each image that ends behind the tensor's first byte, if there is one, decides
    const __int128 begin = (__int128)(uintptr_t)t->data;
    for (int i = 0; i < (image ? images : 1); ++i) {
        const __int128 first = at + i * image, before = begin - first - keys;                // its own rows up to before / query end in front of the tensor
        const __int128 j = before < 0 || !query ? 0 : before / query + 1, row = first + j * query;
        if (j < queries && row <= (__int128)(UINTPTR_MAX - keys) && reaches_into(t, (const void *)(uintptr_t)row, (size_t)keys)) return true;
    }
    return false;
}

}  // namespace dnb

using namespace dnb;

extern "C" int dnb_attention_plan_create(const dnb_attention_desc *desc, dnb_attention_plan **plan)
{
    if (!desc || !plan) DNB_FAIL(DNB_EINVAL, "attention: null argument");
    *plan = nullptr;
    const dnb_attention_desc &d = *desc;
    if (d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads) DNB_FAIL(DNB_EINVAL, "attention: %d query heads for %d key heads", d.heads, d.kv_heads);
    if (d.head_dim < 8 || d.head_dim % 8) DNB_FAIL(DNB_EINVAL, "attention: heads of %d channels (need a multiple of 8)", d.head_dim);
    if (d.head_dim > 128) DNB_FAIL(DNB_EUNSUPPORTED, "attention: heads of %d channels (at most 128)", d.head_dim);
    if ((long long)d.heads * d.head_dim >= 1LL << 24) DNB_FAIL(DNB_EUNSUPPORTED, "attention: %d heads of %d channels", d.heads, d.head_dim);
    if (!isfinite(d.scale * LOG2E)) DNB_FAIL(DNB_EINVAL, "attention: scale %g (times log2 e it has to be finite)", (double)d.scale);   // exponentials are taken to base 2
    // Without a device the plan still checks the arguments of its calls, and then refuses them.
    int device = -1, *status = nullptr;
    if (cudaGetDevice(&device) != cudaSuccess || cudaMalloc(&status, sizeof(int)) != cudaSuccess) {
        const cudaError_t e = cudaGetLastError();
        if (e != cudaErrorNoDevice && e != cudaErrorInsufficientDriver) DNB_FAIL(DNB_ECUDA, "attention: no memory for the plan's status word: %s", cudaGetErrorString(e));
        device = -1;
        status = nullptr;
    }
    const cudaError_t cleared = status ? cudaMemset(status, 0, sizeof(int)) : cudaSuccess;
    dnb_attention_plan *p = cleared == cudaSuccess ? new (std::nothrow) dnb_attention_plan() : nullptr;
    if (!p) {
        cudaFree(status);
        DNB_CUDA(cleared);
        DNB_FAIL(DNB_ENOMEM, "attention: no memory for the plan");
    }
    p->d = d;
    if (p->d.scale == 0.f) p->d.scale = 1.f / sqrtf((float)d.head_dim);
    p->device = device;
    p->status = status;
    p->kernel.store("none", std::memory_order_relaxed);
    *plan = p;
    return DNB_OK;
}

extern "C" void dnb_attention_plan_destroy(dnb_attention_plan *p)
{
    if (!p) return;
    if (p->status) cudaFree(p->status);
    delete p;
}

extern "C" int dnb_attention_forward(dnb_attention_plan *p, const dnb_tensor *q, const dnb_tensor *k, const dnb_tensor *v, const dnb_attention_mask *mask,
                                     const dnb_tensor *y, void *stream)
{
    if (!p) DNB_FAIL(DNB_EINVAL, "attention: null plan");
    DNB_TRY(check_tensor(q, "attention queries"));
    DNB_TRY(check_tensor(k, "attention keys"));
    DNB_TRY(check_tensor(v, "attention values"));
    DNB_TRY(check_tensor(y, "attention output"));
    for (const dnb_tensor *t : {q, k, v, y})
        if (t->layout != DNB_NHWC || t->dtype != q->dtype) DNB_FAIL(DNB_EINVAL, "attention: tensors must be channels-last and of one dtype");
    const dnb_attention_desc &d = p->d;
    if (q->c != d.heads * d.head_dim) DNB_FAIL(DNB_EINVAL, "attention: %d query channels for %d heads of %d", q->c, d.heads, d.head_dim);
    if (k->c != d.kv_heads * d.head_dim) DNB_FAIL(DNB_EINVAL, "attention: %d key channels for %d heads of %d", k->c, d.kv_heads, d.head_dim);
    if (v->n != k->n || v->c != k->c || v->h != k->h || v->w != k->w) DNB_FAIL(DNB_EINVAL, "attention: keys and values differ in extents");
    if (y->n != q->n || y->c != q->c || y->h != q->h || y->w != q->w) DNB_FAIL(DNB_EINVAL, "attention: queries and output differ in extents");
    if (k->n != q->n && k->n != 1) DNB_FAIL(DNB_EINVAL, "attention: keys of %d images for queries of %d (one for all, or one each)", k->n, q->n);
    for (const dnb_tensor *t : {q, k, v})
        if (share_memory(t, y)) DNB_FAIL(DNB_EINVAL, "attention: the output is an input's memory");
    if ((long long)q->h * q->w > 1LL << 30 || (long long)k->h * k->w > 1LL << 30) DNB_FAIL(DNB_EUNSUPPORTED, "attention: more than 2^30 tokens an image");
    AttnArgs a = {};
    a.q = q->data; a.k = k->data; a.v = v->data; a.y = y->data;
    a.n = q->n; a.kn = k->n;
    a.lq = q->h * q->w; a.lk = k->h * k->w;
    a.heads = d.heads; a.kv_heads = d.kv_heads; a.group = d.heads / d.kv_heads; a.d = d.head_dim;
    a.qp = q->cpitch; a.kp = k->cpitch; a.vp = v->cpitch; a.yp = y->cpitch;
    a.scale = d.scale;
    if (mask) {
        if ((uintptr_t)mask->lengths % 4) DNB_FAIL(DNB_EINVAL, "attention: lengths must be 4-byte aligned");
        if (mask->mask && (mask->image_stride < 0 || mask->query_stride < 0)) DNB_FAIL(DNB_EINVAL, "attention: negative strides of the mask");
        if (mask->lengths && reaches_into(y, mask->lengths, (size_t)q->n * 4)) DNB_FAIL(DNB_EINVAL, "attention: the output is the lengths' memory");
        if (mask->mask && reaches_into_mask(y, mask, a.n, a.lq, a.lk)) DNB_FAIL(DNB_EINVAL, "attention: the output is the mask's memory");
        a.lengths = mask->lengths;
        a.mask = mask->mask; a.mask_image = mask->image_stride; a.mask_query = a.lq > 1 ? mask->query_stride : 0;   // one query: one mask for all of them
    }
    a.status = p->status; a.debug = p->debug;
    // a poll of a barrier that does not come takes about 2900 clocks: the hardware suspends the thread meanwhile
    const long long polls = (p->wait_limit ? p->wait_limit : WAIT_LIMIT_CYCLES) / 2048 + 1;
    a.polls = polls > 0x7fffffff ? 0x7fffffff : (int)polls;
    if (p->device < 0) DNB_FAIL(DNB_ECUDA, "attention: the plan was made without a CUDA device");
    DNB_TRY(check_current_device(p->device, "attention"));
    if (attention_rows_covers(a)) {
        p->kernel.store(q->dtype == DNB_F32 ? "rows_f32" : "rows_bf16", std::memory_order_relaxed);
        return launch_attention_rows(a, q->dtype, (cudaStream_t)stream);
    }
    if (attention_f32_tc_covers(a, q->dtype)) {
        p->kernel.store("tc_f32", std::memory_order_relaxed);
        return launch_attention_f32_tc(a, (cudaStream_t)stream);
    }
    if (attention_tc_covers(a, q->dtype)) {
        p->kernel.store("tc_bf16", std::memory_order_relaxed);
        return launch_attention_tc(a, (cudaStream_t)stream);
    }
    p->kernel.store("simple", std::memory_order_relaxed);
    return launch_attention_simple(a, q->dtype, (cudaStream_t)stream);
}

extern "C" int dnb_attention_plan_check_status(dnb_attention_plan *p)
{
    if (!p) DNB_FAIL(DNB_EINVAL, "attention: null plan");
    if (!p->status) return DNB_OK;
    int v = 0;
    DNB_CUDA(cudaMemcpy(&v, p->status, sizeof(int), cudaMemcpyDeviceToHost));
    if (v) {
        cudaMemset(p->status, 0, sizeof(int));
        DNB_FAIL(DNB_ETIMEOUT, "attention: a device-side wait expired (code %d)", v);
    }
    return DNB_OK;
}

extern "C" int dnb_attention_plan_set_diagnostics(dnb_attention_plan *p, long long wait_limit_cycles, int debug_bits)
{
    if (!p || wait_limit_cycles < 0 || (debug_bits & ~32)) DNB_FAIL(DNB_EINVAL, "attention: diagnostics");
    p->wait_limit = wait_limit_cycles;
    p->debug = debug_bits;
    return DNB_OK;
}

extern "C" const char *dnb_attention_plan_kernel(const dnb_attention_plan *p) { return p ? p->kernel.load(std::memory_order_relaxed) : "none"; }
