// PAGED_PLAN and ROPE_AXES / ROPE_AXES_STORE (include/scrapgpu/hip_ops.h) on gfx950.
#include "serving.h"

#include <hip/hip_fp16.h>

#include <algorithm>
#include <cstdio>

namespace sgk {
namespace {

// ---- PAGED_PLAN ---------------------------------------------------------------------------------
//
// Everything follows from three prefix sums over the requests (new tokens, new pages, pages that
// come back): who enters (the sums up to the first request that does not fit), the token ranges, and
// for the a-th new page of the step which free page it is (entry have - 1 - a of the pool with the
// returned pages on top). So one launch does it: every work-group forms the sums of all requests in
// LDS (a few loads and one scan; a request list is at most 2048 long), then takes its share of the
// tokens, the new pages and the returned pages. No work-group reads what another writes: a token
// finds its page in the table only below its request's old pages, which nobody writes, and otherwise
// in the pool below `free`, which nobody writes either, or in an ended request's table row.
// kv_len and left may lie over past and free, so they and q_start are written by the last
// work-group to arrive, when all have read their inputs.
//
// Bound: latency (two dependent loads, a scan, a search, one more load, the store; the bytes are a
// few hundred KB at most). 64 requests of one new token 6.6 us a call, 256 of up to 150 new tokens 7.5;
// the host's side of any op takes 3.5 to 4.

constexpr int kPlanThreads = 256;
constexpr uint32_t kMany = 1u << 30; // sums stop here: larger ones never fit

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
    return min(a + b, kMany);
}

// the last index i < n with at[i] <= x (at[0] = 0; ascending)
__device__ __forceinline__ int last_not_above(const uint32_t * at, int n, uint32_t x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanLaunch a) {
    // sums over the requests before b: new tokens, new pages, returned pages
    __shared__ uint32_t tok[kPlanRequests + 1], need[kPlanRequests + 1], back[kPlanRequests + 1];
    __shared__ int past[kPlanRequests];
    __shared__ uint32_t part[3][kPlanThreads / 64];
    __shared__ uint32_t first_bad, refused_long;
    __shared__ bool last;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int page = 1 << a.shift;
    const int free_n = min(max(a.free_in[0], 0), a.P);
    const uint32_t room = (uint32_t) a.W << a.shift;
    if (t == 0) {
        first_bad = (uint32_t) a.B;
        refused_long = 0;
    }
    uint32_t carry[3] = {0, 0, 0};
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
        const int b = b0 + t;
        uint32_t v[3] = {0, 0, 0};
        if (b < a.B) {
            const int p = min(max(a.past[b], 0), (int) room), f = a.fresh[b];
            past[b] = p;
            const uint32_t old = (uint32_t) (p + page - 1) >> a.shift;
            if (f < 0) v[2] = old;
            else if ((uint32_t) f > room - (uint32_t) p) v[0] = 0; // longer than a table row
            else if (f > 0) {
                v[0] = (uint32_t) f;
                v[1] = ((uint32_t) (p + f + page - 1) >> a.shift) - old;
            }
        }
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = __shfl_up(v[i], d);
                if (lane >= d) v[i] = add_sat(v[i], o);
            }
        if (lane == 63) {
#pragma unroll
            for (int i = 0; i < 3; ++i) part[i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            uint32_t before = carry[i];
            for (int w = 0; w < wave; ++w) before = add_sat(before, part[i][w]);
            v[i] = add_sat(v[i], before);
            for (int w = 0; w < kPlanThreads / 64; ++w) carry[i] = add_sat(carry[i], part[i][w]);
        }
        if (b < a.B) {
            tok[b + 1] = v[0];
            need[b + 1] = v[1];
            back[b + 1] = v[2];
        }
        __syncthreads();
    }
    if (t == 0) tok[0] = need[0] = back[0] = 0;
    __syncthreads();
    const uint32_t have = min((uint32_t) free_n + back[a.B], kMany);
    for (int b = t; b < a.B; b += kPlanThreads)
        if (tok[b + 1] > tok[b] && (tok[b + 1] > (uint32_t) a.T || need[b + 1] > have)) atomicMin(&first_bad, (uint32_t) b);
    __syncthreads();
    // from the first request that does not fit on, none enters
    const uint32_t n_tok = tok[first_bad], n_need = need[first_bad], n_back = back[a.B];
    const int n_in = (int) first_bad;

    // entry i of the pool with the returned pages on top
    const auto page_at = [&](int64_t i) {
        if (i < 0) return -1;
        if (i < free_n) return a.pool[i];
        const uint32_t r = (uint32_t) (i - free_n);
        const int b = last_not_above(back, a.B, r);
        return a.table[b * a.t_s1 + min(r - back[b], (uint32_t) a.W - 1)];
    };
    const int stride = gridDim.x * kPlanThreads, me = blockIdx.x * kPlanThreads + t;
    for (int i = me; i < a.T; i += stride) {
        int pos = 0, slot = -1;
        if ((uint32_t) i < n_tok) {
            const int b = last_not_above(tok, n_in, (uint32_t) i);
            pos = past[b] + (i - (int) tok[b]);
            const int j = pos >> a.shift, old = (past[b] + page - 1) >> a.shift;
            const int pg = j < old ? a.table[b * a.t_s1 + j] : page_at((int64_t) have - 1 - need[b] - (j - old));
            slot = pg < 0 || pg > (0x7FFFFFFF >> a.shift) ? -1 : (pg << a.shift) + (pos & (page - 1));
        }
        a.pos[i] = pos;
        a.slots[i] = slot;
    }
    for (uint32_t i = (uint32_t) me; i < n_need; i += (uint32_t) stride) {
        const int b = last_not_above(need, n_in, i);
        const int j = ((past[b] + page - 1) >> a.shift) + (int) (i - need[b]);
        if (j < a.W) a.table[b * a.t_s1 + j] = page_at((int64_t) have - 1 - i);
    }
    for (uint32_t i = (uint32_t) me; i < n_back; i += (uint32_t) stride)
        if (free_n + (int64_t) i < a.P) a.pool[free_n + i] = page_at(free_n + (int64_t) i);

    // the last work-group has the others' arrivals behind it, so their reads of past, fresh and free
    __syncthreads();
    if (t == 0) {
        last = gridDim.x == 1 || atomicAdd(a.arrive, 1u) == gridDim.x - 1;
        if (last && gridDim.x > 1) *a.arrive = 0;
    }
    __syncthreads();
    if (!last) return;
    uint32_t refused = 0;
    for (int b = t; b < a.B; b += kPlanThreads) {
        const int f = a.fresh[b];
        const uint32_t n = b < n_in ? tok[b + 1] - tok[b] : 0;
        refused += f > 0 && n == 0;
        a.q_start[b] = (int) min(tok[b], n_tok);
        a.kv_len[b] = f < 0 ? 0 : past[b] + (int) n;
    }
    if (refused) atomicAdd(&refused_long, refused);
    __syncthreads();
    if (t == 0) {
        a.q_start[a.B] = (int) n_tok;
        a.left[0] = (int) (have - n_need);
        a.left[1] = (int) refused_long;
    }
}

} // namespace

hipError_t launch_paged_plan(const PlanLaunch & p, int cu_count, hipStream_t stream) {
    if (p.B < 1 || p.B > kPlanRequests || p.T < 1) return hipErrorInvalidValue;
    // a work-group per 256 tokens
    const int grid = std::min((p.T + kPlanThreads - 1) / kPlanThreads, cu_count);
    std::snprintf(last_form().form, sizeof(last_form().form), "paged plan");
    last_form().grid = (uint64_t) grid;
    k_paged_plan<<<dim3((unsigned) grid), dim3(kPlanThreads), 0, stream>>>(p);
    return hipGetLastError();
}

namespace {

// ---- ROPE_AXES, ROPE_AXES_STORE -------------------------------------------------------------------
//
// A thread owns V pairs of elements (or 2 V copied ones) of one token and goes over heads of q, k
// and v with them, so an angle's sine and cosine are formed once per token and thread. The angle is
// formed in whole numbers: position times 2^64 turns mod 2^64 is the exact fraction of a turn for
// any 32-bit position (an f32 product of position and frequency is off by 2^-24 of the whole angle,
// 1e-3 at position 16384); its top 32 bits, as a signed number of half turns, go through sincospi.
//
// Bound: the bytes of q, k, v in and out. 4099 tokens of 28/4 heads of 128, f32 into bf16: 113 MB in
// 25 us, 4.5 TB/s (a large copy reaches 5.0); 5329 of 16 heads of 80, bf16: 27 MB in 9.4 us, 2.9 TB/s,
// of which the sines and the start of the launch take about half; 8 tokens 4 to 5 us.

template <int TY> struct Elem;
template <> struct Elem<F32> {
    typedef float type;
    static __device__ float to(float v) { return v; }
    static __device__ float from(float v) { return v; }
};
template <> struct Elem<F16> {
    typedef _Float16 type;
    static __device__ float to(_Float16 v) { return (float) v; }
    static __device__ _Float16 from(float v) { return (_Float16) v; }
};
template <> struct Elem<BF16> {
    typedef __bf16 type;
    static __device__ float to(__bf16 v) { return (float) v; }
    static __device__ __bf16 from(float v) { return (__bf16) v; }
};

template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
    T e[N];
};

// a thread's 2 V elements: V at `first`, V at `second` (apart by half the turned elements, or by V)
template <int TY, int V> struct Pairs {
    typedef typename Elem<TY>::type T;
    Pack<T, V> a, b;
    __device__ __forceinline__ void load(const uint8_t * p, int first, int second) {
        const T * e = reinterpret_cast<const T *>(p);
        a = *reinterpret_cast<const Pack<T, V> *>(e + first);
        b = *reinterpret_cast<const Pack<T, V> *>(e + second);
    }
};
template <int TY, int V>
__device__ __forceinline__ void store_pairs(uint8_t * p, int first, int second, const float * x, const float * z) {
    typedef typename Elem<TY>::type T;
    T * e = reinterpret_cast<T *>(p);
    Pack<T, V> a, b;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        a.e[i] = Elem<TY>::from(x[i]);
        b.e[i] = Elem<TY>::from(z[i]);
    }
    *reinterpret_cast<Pack<T, V> *>(e + first) = a;
    *reinterpret_cast<Pack<T, V> *>(e + second) = b;
}

template <int V>
__device__ __forceinline__ void store_any(int type, uint8_t * p, int first, int second, const float * x, const float * z) {
    if (type == F32) store_pairs<F32, V>(p, first, second, x, z);
    else if (type == F16) store_pairs<F16, V>(p, first, second, x, z);
    else store_pairs<BF16, V>(p, first, second, x, z);
}

template <int IN, int V, bool ADJ>
__global__ __launch_bounds__(256) void k_rope(RopeLaunch a, int chunks, int per_block_heads) {
    const int id = blockIdx.x * 256 + threadIdx.x;
    const int t = id / chunks, c = id - t * chunks;
    if (t >= a.T) return;
    const int turned = a.n_dims / (2 * V); // chunks of pairs; the rest are copied
    const bool turns = c < turned;
    int first, second;
    if (turns) {
        first = ADJ ? 2 * V * c : V * c;
        second = ADJ ? first + V : first + a.n_dims / 2;
    } else {
        first = a.n_dims + 2 * V * (c - turned);
        second = first + V;
    }
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        cs[i] = 1.0f;
        sn[i] = 0.0f;
        if (turns) {
            const int pair = V * c + i;
            const int64_t pos = a.pos[t * a.p_s1 + a.axis[pair]];
            const int32_t half_turns = (int32_t) (((uint64_t) pos * a.turn[pair]) >> 32);
            sincospif((float) half_turns * 0x1p-31f, &sn[i], &cs[i]);
        }
    }
    const int slot = a.Hk ? a.slots[t] : 0;
    const bool keep = slot >= 0 && slot < a.n_slots;
    const int64_t place = slot & ((1 << a.shift) - 1), pg = slot >> a.shift;
    const int h0 = blockIdx.y * per_block_heads, h1 = min(h0 + per_block_heads, a.Hq + 2 * a.Hk);
    // (heads in batches whose loads are issued before the first store, which they might alias)
    constexpr int BATCH = 6;
    for (int hb = h0; hb < h1; hb += BATCH) {
        Pairs<IN, V> in[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int h = min(hb + k, h1 - 1);
            const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
            const int hk = is_v ? h - a.Hq - a.Hk : h - a.Hq;
            in[k].load(is_q ? a.q + h * a.q_s1 + t * a.q_s2 : is_v ? a.v + hk * a.v_s1 + t * a.v_s2 : a.k + hk * a.k_s1 + t * a.k_s2, first, second);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int h = hb + k;
            if (h >= h1) break;
            const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
            if (!is_q && !keep) break;
            const int hk = is_v ? h - a.Hq - a.Hk : h - a.Hq;
            float x[V], z[V], u[V], w[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[i] = Elem<IN>::to(in[k].a.e[i]);
                z[i] = Elem<IN>::to(in[k].b.e[i]);
            }
            if (is_v || !turns) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u[i] = x[i];
                    w[i] = z[i];
                }
            } else if (ADJ) {
                float y[2 * V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float p = 2 * i < V ? x[(2 * i) % V] : z[(2 * i) % V], q = 2 * i + 1 < V ? x[(2 * i + 1) % V] : z[(2 * i + 1) % V];
                    y[2 * i] = p * cs[i] - q * sn[i];
                    y[2 * i + 1] = p * sn[i] + q * cs[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u[i] = y[i];
                    w[i] = y[V + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u[i] = x[i] * cs[i] - z[i] * sn[i];
                    w[i] = x[i] * sn[i] + z[i] * cs[i];
                }
            }
            if (is_q) store_any<V>(a.out_type, a.y + h * a.y_s1 + t * a.y_s2, first, second, u, w);
            else if (is_v) store_any<V>(a.cache_type, a.vc + place * a.vc_s1 + hk * a.vc_s2 + pg * a.vc_s3, first, second, u, w);
            else store_any<V>(a.cache_type, a.kc + place * a.kc_s1 + hk * a.kc_s2 + pg * a.kc_s3, first, second, u, w);
        }
    }
}

int bytes_of(int type) {
    return type == F32 ? 4 : 2;
}

} // namespace

hipError_t launch_rope(const RopeLaunch & r, int cu_count, hipStream_t stream) {
    if (r.T < 1 || r.D % 2 != 0 || r.n_dims > 256 || r.n_dims > r.D) return hipErrorInvalidValue;
    // V pairs a thread: 4 where shape and alignment allow it, also for 16-bit types, whose loads are 8 bytes
    // then (with 8 pairs a thread has 8 sines to form: 30000 tokens of 8 heads of 256 in bf16 40 us, 53 with
    // 8; 5329 of 16 of 80 9.7, 11.4 with 8)
    const auto fits = [&](int v) {
        if (r.n_dims % (2 * v) != 0 || (r.D - r.n_dims) % (2 * v) != 0) return false;
        uint64_t in = reinterpret_cast<uint64_t>(r.q) | (r.Hq > 1 ? r.q_s1 : 0) | (r.T > 1 ? r.q_s2 : 0);
        uint64_t out = reinterpret_cast<uint64_t>(r.y) | (r.Hq > 1 ? r.y_s1 : 0) | (r.T > 1 ? r.y_s2 : 0);
        if (r.Hk) in |= reinterpret_cast<uint64_t>(r.k) | reinterpret_cast<uint64_t>(r.v) | (r.Hk > 1 ? r.k_s1 | r.v_s1 : 0) | (r.T > 1 ? r.k_s2 | r.v_s2 : 0);
        return in % (uint64_t) (v * bytes_of(r.in_type)) == 0 && out % (uint64_t) (v * bytes_of(r.out_type)) == 0;
        // (the caches' strides are multiples of 16 bytes)
    };
    const int V = fits(4) ? 4 : 1;
    const int chunks = r.D / (2 * V), heads = r.Hq + 2 * r.Hk;
    // a launch for as many tokens as 32-bit thread numbers reach (all but a few calls of many GB)
    const int most = 0x7FFFFFFF / chunks;
    last_form().grid = 0;
    for (int64_t t0 = 0; t0 < r.T; t0 += most) {
        RopeLaunch part = r;
        part.T = (int) std::min<int64_t>(most, r.T - t0);
        part.q += t0 * r.q_s2;
        part.y += t0 * r.y_s2;
        part.pos += t0 * r.p_s1;
        if (r.Hk) {
            part.k += t0 * r.k_s2;
            part.v += t0 * r.v_s2;
            part.slots += t0;
        }
        const int64_t blocks = ((int64_t) part.T * chunks + 255) / 256;
        // few tokens: the heads over more work-groups, until each CU has four
        const int64_t split = std::max<int64_t>(1, std::min<int64_t>(heads, 4 * cu_count / blocks));
        const int per = (int) ((heads + split - 1) / split);
        const dim3 grid((unsigned) blocks, (unsigned) ((heads + per - 1) / per));
        std::snprintf(last_form().form, sizeof(last_form().form), "rope v=%d heads=%d", V, per);
        last_form().grid += (uint64_t) grid.x * grid.y;
        const auto go = [&](auto kernel) { kernel<<<grid, dim3(256), 0, stream>>>(part, chunks, per); };
        const auto pick = [&](auto in) {
            constexpr int IN = decltype(in)::value;
            if (V == 4) r.adjacent ? go(k_rope<IN, 4, true>) : go(k_rope<IN, 4, false>);
            else r.adjacent ? go(k_rope<IN, 1, true>) : go(k_rope<IN, 1, false>);
        };
        if (r.in_type == F32) pick(std::integral_constant<int, F32>{});
        else if (r.in_type == F16) pick(std::integral_constant<int, F16>{});
        else pick(std::integral_constant<int, BF16>{});
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

} // namespace sgk
