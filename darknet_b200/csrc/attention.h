// Internal argument blocks of the cross-attention kernels and the plan object.
#pragma once
#include <atomic>

#include "common.h"

struct dnb_attention_plan {
    dnb_attention_desc d;
    int device;
    int *status;            // device word: 0, or the code of the bounded wait that ran out
    long long wait_limit;   // SM clock cycles
    int debug;
    std::atomic<const char *> kernel;   // of the last forward of any thread, for logs and tests
};

namespace dnb {

// One call.  Queries i of image n and head h: row n*lq + i of q, channels h*d ..; keys and values: row (kn == 1 ? 0 : n)*lk + j, channels h/group*d ..
struct AttnArgs {
    const void *q, *k, *v;
    void *y;
    int n, kn, lq, lk;
    int heads, kv_heads, group, d;
    int qp, kp, vp, yp;                     // pitches, elements
    float scale;
    const int32_t *lengths;                 // keys of each image, or null: all
    const uint8_t *mask;                    // or null
    long long mask_image, mask_query;       // its strides, bytes
    int *status;
    int polls;                              // bound of every device-side wait
    int debug;
};

// How many CTAs share the keys of one job (1, 2, 4 or 8: a cluster), as if every image had all its keys.  A wave of CTAs takes its tiles of keys, `start` tiles' time to begin and end, and
// `join` tiles' for each CTA that joins; room[i]: the CTAs of clusters of 2^i that run at once.
int split_keys(long long jobs, int key_tiles, const int room[4], double start, double join);
// room of a kernel of one CTA an SM, asked once a device and slot (0 .. 7)
int cluster_room(const void *kernel, int slot, int threads, size_t smem, int room[4]);

// ---- cross_attention.cu
int launch_attention_simple(const AttnArgs &a, int dtype, cudaStream_t s);

// ---- cross_attention_tc.cu : bf16, on the tensor cores
bool attention_tc_covers(const AttnArgs &a, int dtype);
int launch_attention_tc(const AttnArgs &a, cudaStream_t s);

// ---- cross_attention_rows.cu : up to 16 rows a key head
bool attention_rows_covers(const AttnArgs &a);
int launch_attention_rows(const AttnArgs &a, int dtype, cudaStream_t s);

// ---- cross_attention_f32_tc.cu : f32, on the tensor cores
bool attention_f32_tc_covers(const AttnArgs &a, int dtype);
int launch_attention_f32_tc(const AttnArgs &a, cudaStream_t s);

}  // namespace dnb
