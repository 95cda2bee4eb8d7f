// The serving ops (include/scrapgpu/hip_ops.h): their support rules (serving.cpp) and the launch
// interface of their kernels (paged.hip, attention.hip, attention_decode.hip).
#pragma once

#include "kernels.h"

#include "scrapgpu/hip_ops.h"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sgk {

// PAGED_PLAN over B requests, rows of W table entries (t_s1 entries apart), P pool entries, T tokens
constexpr int kPlanRequests = 2048;
struct PlanLaunch {
    const int32_t *past, *fresh, *free_in;
    int32_t *table, *pool, *left, *q_start, *kv_len, *pos, *slots;
    int64_t t_s1;
    int B, W, P, T;
    int shift;         // page size = 1 << shift
    uint32_t * arrive; // a count that is zero before the launch and left at zero
};
hipError_t launch_paged_plan(const PlanLaunch & p, int cu_count, hipStream_t stream);

// ROPE_AXES (k, v null) and ROPE_AXES_STORE. Strides in bytes: s1 between heads, s2 between tokens;
// the caches' s1 between places, s2 between heads, s3 between pages.
struct RopeLaunch {
    int in_type, out_type, cache_type;
    const uint8_t *q, *k, *v;
    uint8_t *y, *kc, *vc;
    uint64_t q_s1, q_s2, k_s1, k_s2, v_s1, v_s2, y_s1, y_s2;
    uint64_t kc_s1, kc_s2, kc_s3, vc_s1, vc_s2, vc_s3;
    const int32_t *pos, *slots;
    int64_t p_s1;      // elements between tokens' positions
    int64_t n_slots;   // slots of the cache
    int T, Hq, Hk, D, n_dims, shift, adjacent;
    uint64_t turn[128]; // pair i's turns per position, times 2^64
    uint8_t axis[128];
};
hipError_t launch_rope(const RopeLaunch & r, int cu_count, hipStream_t stream);

// ATTENTION_PROMPT / ATTENTION_PAGED. Strides in bytes: q, o: s1 between heads, s2 between tokens;
// k, v: s1 between tokens (places), s2 between heads, s3 between pages.
struct AttnLaunch {
    int dtype, out_type;
    const uint8_t *q, *k, *v;
    uint8_t * o;
    uint64_t q_s1, q_s2, o_s1, o_s2, k_s1, k_s2, k_s3, v_s1, v_s2, v_s3;
    const int32_t * table; // null: prompts
    int64_t t_s1;
    int W, shift, n_pages;
    const int32_t * q_start;
    const int32_t * k_at; // prompts: k_start (B + 1); paged: kv_len (B)
    int B, T, Tk, Hq, Hk, G, D;
    float scale;
    int causal, max_query;
    bool paged; // (known before the table's address)
};
// how a launch is cut; the same for every call about one launch
struct AttnShape {
    bool few;       // the kernel for few rows, else tiles of 128
    int nb;         // few rows: blocks of 16 of them in registers
    int tiles;      // tiles of all requests at most
    int want;       // pieces of all requests' keys (tiles' keys) wished for per key head; 0: none
    int idle;       // few rows: work-groups to each key head beyond the pieces there can be
    size_t scratch; // bytes
};
// `lean`: partial sums within 32 MiB (fewer pieces; results differ in rounding)
AttnShape attention_shape(const AttnLaunch & a, int cu_count, bool lean);
int64_t attention_groups(const AttnLaunch & a, const AttnShape & s); // work-groups of the launch
hipError_t launch_attention(const AttnLaunch & a, uint8_t * scratch, uint32_t * arrive, int cu_count, bool lean, hipStream_t stream);

} // namespace sgk

// One serving op as its descriptors describe it: the launch arguments without addresses, and where
// each tensor's address goes.
struct ServingOp {
    int op = 0;
    bool empty = false; // no token: nothing to launch
    sgk::PlanLaunch plan;
    sgk::RopeLaunch rope;
    sgk::AttnLaunch attn;
    struct Slot {
        const scrapgpu_tensor_desc * t;
        const char * what;
        void * at; // a pointer member of plan / rope / attn
    } slots[12];
    int n_slots = 0;
    double bytes = 0, flops = 0; // for the event profiler: what the tensors' shapes say (the lengths are on the device)
};

bool is_serving_op(int op);
// the support rule; fills `out` unless it is null. A status other than OK carries its reason in *reason.
scrapgpu_status serving_rule(const scrapgpu_op_desc * desc, ServingOp * out, const char ** reason);
