// What the two attention kernels (attention.hip: tiles of 128 rows; attention_decode.hip: few rows)
// share on the device.
//
// Both form S^T = K Q^T and O^T = V^T P^T, so that a query row is a column of the matrix units'
// results: a lane holds scores of one row only, its maximum, sum and rescaling are plain numbers of
// the lane, and the scores, rounded to 16 bits, are already the second product's operand (the order
// of the keys inside a step is permuted the same way on both sides). A "row" is one query head of
// one token; the G query heads that share a key head are rows of one tile (row = token * G + head),
// so each key and value is read once for all of them.
#pragma once

#include "serving.h"

namespace sgk {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -1e30f; // the running maximum before any key (finite: no Inf - Inf)
// A row's sums are relative to a maximum that may lag behind the true one: it is brought up to date,
// and the sums with it, only when it lags by more than kLag (log2).
constexpr float kLag = 6.0f;
// What sums relative to one maximum are worth relative to another; never 0, so that infinite sums stay
// infinite. What is left of a finite one at least is 2^-149 of it: f32 weights lie that far apart near zero
// (a select on infinite sums instead: 512 tokens over 6000 beside 15 single ones, 111 -> 123 us).
__device__ __forceinline__ float decay(float from, float to) {
    return fmaxf(__builtin_amdgcn_exp2f(from - to), 0x1p-149f);
}
// F16 weights are scaled by 2^8 (with kLag: at most 2^14 of 65504), so that weights down to 2^-22 of
// the largest stay normal numbers; the scale cancels in the division by the sum. BF16 needs none.
template <int DT> constexpr float kLift = DT == F16 ? 8.0f : 0.0f;

// Two f32 weights as 16-bit elements, and their sum added to `total`. The sum is that of the rounded
// weights (each exact in f32): the division by it takes the rounding's bias out again, so F16 may cut
// off (one instruction; its error is then as large as rounding's), BF16 rounds to nearest.
template <int DT>
__device__ __forceinline__ uint32_t round2(float a, float b, float & total) {
    if constexpr (DT == F16) {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        const auto t = __builtin_amdgcn_cvt_pkrtz(a, b);
        const pair v = __builtin_bit_cast(pair, t);
        total = __builtin_amdgcn_fdot2(v, pair{(_Float16) 1.0f, (_Float16) 1.0f}, total, false);
        return __builtin_bit_cast(uint32_t, v);
    } else {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        const pair v = {(__bf16) a, (__bf16) b};
        total = __builtin_amdgcn_fdot2_f32_bf16(v, pair{(__bf16) 1.0f, (__bf16) 1.0f}, total, false);
        return __builtin_bit_cast(uint32_t, v);
    }
}
// Elements between rows of a kernel that computes with DW of them: a power of two, which permutes well
constexpr int padded(int DW) {
    return DW == 96 ? 128 : DW;
}

// the kernel for few rows: work-groups per CU that the registers are held to (NB blocks of 16 rows)
constexpr int resident(int DP, int NB) {
    return DP * NB <= 64 ? 4 : DP * NB <= 256 && DP < 256 ? 2 : 1;
}

// A weight as the sum of N terms of the type, each what the ones before leave. F32 results: two of F16 (22
// bits), three of BF16 (24; two leave errors of 4e-6 of the result, where f32 sums leave 3e-7). 16-bit results
// of few rows: two (BF16: 16 bits). What a weight below 2^-22 of the largest loses in F16 (below 2^-14, lifted)
// is under 2^-32 of the largest.
template <int DT> constexpr int kTerms = DT == F16 ? 2 : 3;
template <int DT, int N>
__device__ __forceinline__ void split(float a, float b, uint32_t (&term)[N]) {
    constexpr uint32_t M = DT == F16 ? 0xFFFFE000u : 0xFFFF0000u;
    const float x = __uint_as_float(__float_as_uint(a) & M), y = __uint_as_float(__float_as_uint(b) & M);
    const float r = a - x, t = b - y;
    if constexpr (DT == F16) {
        static_assert(N == 2);
        const auto u = __builtin_amdgcn_cvt_pkrtz(x, y), v = __builtin_amdgcn_cvt_pkrtz(r, t);
        term[0] = __builtin_bit_cast(uint32_t, u);
        term[1] = __builtin_bit_cast(uint32_t, v);
    } else {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        term[0] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        if constexpr (N == 2) {
            const pair v = {(__bf16) r, (__bf16) t};
            term[1] = __builtin_bit_cast(uint32_t, v);
        } else {
            const pair v = {(__bf16) (r - __uint_as_float(__float_as_uint(r) & M)), (__bf16) (t - __uint_as_float(__float_as_uint(t) & M))};
            term[1] = __builtin_amdgcn_perm(__float_as_uint(t), __float_as_uint(r), 0x07060302u);
            term[2] = __builtin_bit_cast(uint32_t, v);
        }
    }
}

// the value of the lower and of the upper half-wave's lane, in both
__device__ __forceinline__ float2 both_halves(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const uint32_t lo = r[0], hi = r[1]; // (a bit cast of a vector's element reads the first one)
    return make_float2(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float max_halves(float v) {
    const float2 r = both_halves(v);
    return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float sum_halves(float v) {
    const float2 r = both_halves(v);
    return r.x + r.y;
}

// 16 bytes a lane from base + off straight into LDS, lane l's at lds + 16 l (base, lds: one for the
// wave). Written out because the compiler, which knows the builtin's writes to LDS, waits for all of
// them before any transposing read, so also for those just asked for: it must not know, and the
// kernels wait themselves. (No vector register is written.)
__device__ __forceinline__ void load_lds16(const uint8_t * base, uint32_t off, uint8_t * lds) {
    const uint32_t at = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t *) lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(base) : "memory", "m0");
}

// the same for bytes that nobody reads again
__device__ __forceinline__ void load_lds16_once(const uint8_t * base, uint32_t off, uint8_t * lds) {
    const uint32_t at = (uint32_t) (uintptr_t) (__attribute__((address_space(3))) uint8_t *) lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(at), "v"(off), "s"(base) : "memory", "m0");
}

// 4 elements of one column of four rows of LDS (see the kernels' V operands)
__device__ __forceinline__ s16x4 read_column4(const uint8_t * p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *) p);
}

// the request's token range, inside the tensor whatever the starts say (the first starts at 0)
__device__ __forceinline__ int2 range_of(const int32_t * start, int b, int n) {
    const int lo = b == 0 ? 0 : min(max(start[b], 0), n);
    return make_int2(lo, max(lo, min(start[b + 1], n)));
}

// scores to log2 of weights; the scale's sign is in q. Never 0, so that a hidden score, -Inf, stays it.
__device__ __forceinline__ float weight_scale(const AttnLaunch & a) {
    return fmaxf(fabsf(a.scale) * 1.44269504088896341f, 1e-37f);
}

// Zeros for the tokens from `first` on, which belong to no request. The work-groups that find nothing else to do share them (this is
// the `turn`-th of `groups` to each key head): a wave writes as many rows at a time as its lanes hold 16-byte chunks
// of, consecutive waves consecutive ones. A recorded step has places for more tokens than live: 64 tokens over up
// to 8000 keys, of 64 places 199 us, of 8192 211.
__device__ __forceinline__ void zero_rest(const AttnLaunch & a, int first, int kvh, int turn, int groups) {
    if (first >= a.T) return;
    const uint32_t per = a.out_type == F32 ? a.D / 4 : a.D / 8; // chunks of a row: at most 64
    const uint32_t lane = threadIdx.x & 63, rows = 64 / per, waves = blockDim.x / 64;
    const uint32_t step = (uint32_t) (groups * a.Hk) * waves * rows, r = ((uint32_t) (turn * a.Hk + kvh) * waves + threadIdx.x / 64) * rows + lane / per;
    const int64_t step_t = step / (uint32_t) a.Hq;
    const int step_h = step % (uint32_t) a.Hq;
    int64_t t = (int64_t) first + r / (uint32_t) a.Hq;
    int h = r % (uint32_t) a.Hq;
    if (lane >= rows * per) return;
    while (t < a.T) {
        *reinterpret_cast<u32x4 *>(a.o + t * a.o_s2 + h * a.o_s1 + 16 * (lane % per)) = u32x4{0, 0, 0, 0};
        t += step_t;
        h += step_h;
        if (h >= a.Hq) {
            h -= a.Hq;
            ++t;
        }
    }
}

// 4 consecutive elements of an output row
template <int DT, bool OUT32>
__device__ __forceinline__ void store4(uint8_t * row, int d, float a, float b, float c, float e) {
    if constexpr (OUT32) {
        *reinterpret_cast<f32x4 *>(row + 4 * d) = f32x4{a, b, c, e};
    } else if constexpr (DT == F16) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<f16x4 *>(row + 2 * d) = f16x4{(_Float16) a, (_Float16) b, (_Float16) c, (_Float16) e};
    } else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<bf16x4 *>(row + 2 * d) = bf16x4{(__bf16) a, (__bf16) b, (__bf16) c, (__bf16) e};
    }
}

// Inf and NaN among values that some rows of a step do not see: a weight of 0 times one of them is
// NaN, which would reach rows that must not know of it. Such steps look through their values first
// (16 bytes of LDS at a time); where there are any, each row that sees one adds it to its sums by
// itself, and zero takes its place before the product. (Values that all rows see go into the product as
// they are: see settle.)
template <int DT>
__device__ __forceinline__ bool has_nonfinite(u32x4 w) {
    constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (w[i] & E) == E || (w[i] & (E << 16)) == (E << 16);
    return any;
}
template <int DT>
__device__ __forceinline__ u32x4 only_finite(u32x4 w) {
    constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = ((w[i] & E) == E ? 0 : w[i] & 0xFFFFu) | ((w[i] & (E << 16)) == (E << 16) ? 0 : w[i] & 0xFFFF0000u);
    return w;
}
// the f32 value of 16 bits that are Inf or NaN
template <int DT>
__device__ __forceinline__ float nonfinite(uint32_t h) {
    constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
    return __uint_as_float((h & 0x8000u) << 16 | 0x7F800000u | ((h & (0x7FFFu & ~E)) != 0 ? 0x400000u : 0));
}
// calls add(element, value) for each Inf or NaN of each lane's 16 bytes, one after the other, in all
// lanes alike; `at`: the lane's first element
template <int DT, typename F>
__device__ __forceinline__ void each_nonfinite(u32x4 w, int at, F add) {
    constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
    uint64_t lanes = __ballot(has_nonfinite<DT>(w));
    while (lanes != 0) {
        const int l = __builtin_ctzll(lanes);
        lanes &= lanes - 1;
        const int first = __builtin_amdgcn_readlane(at, l);
        const uint32_t x[4] = {(uint32_t) __builtin_amdgcn_readlane(w[0], l), (uint32_t) __builtin_amdgcn_readlane(w[1], l), (uint32_t) __builtin_amdgcn_readlane(w[2], l),
                               (uint32_t) __builtin_amdgcn_readlane(w[3], l)};
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const uint32_t h = (i < 2 ? x[0] : i < 4 ? x[1] : i < 6 ? x[2] : x[3]) >> (16 * (i & 1)) & 0xFFFFu;
            if ((h & E) != E) continue;
            add(first + i, nonfinite<DT>(h));
        }
    }
}

// Seen values that are infinite make a result infinite however small their weight, but a weight, or a
// term of it, that rounds to 0 makes it NaN. So a wave whose sums hold a NaN goes over the values of its
// keys once more: the Inf and NaN that a row sees are all that a sum that came out as NaN is made of (where
// there are none, it stays NaN). Looking through every step's values beforehand would cost every call.
//
// That is as much work whether a few values are infinite or all: of keys that all rows see, a lane sums
// the Inf and NaN of its 16 bytes (keys from .. to - 1, at row_of(key)), and the sums go to the rows, add(element, sum).
template <int DT> struct NonfiniteSum {
    float sum[8] = {};
    template <int DP, typename P> __device__ __forceinline__ void take(int from, int to, int D, P row_of) {
        constexpr int NC = DP / 8;
        constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
        const int lane = threadIdx.x & 63, c = lane % NC;
#pragma unroll 1
        for (int k = from; k < to; k += 64 / NC) {
            const int key = k + lane / NC;
            u32x4 v = {0, 0, 0, 0};
            if (key < to && 8 * c < D) v = *reinterpret_cast<const u32x4 *>(row_of(key) + 16 * c);
            if (!__any(has_nonfinite<DT>(v))) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t h = v[i / 2] >> (16 * (i & 1)) & 0xFFFFu;
                sum[i] += (h & E) == E ? nonfinite<DT>(h) : 0.0f;
            }
        }
    }
    template <int DP, typename F> __device__ __forceinline__ void give(F add) {
        bool some = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) some |= sum[i] != 0.0f;
        uint64_t lanes = __ballot(some);
        while (lanes != 0) {
            const int l = __builtin_ctzll(lanes);
            lanes &= lanes - 1;
#pragma unroll
            for (int i = 0; i < 8; ++i) add(8 * (l % (DP / 8)) + i, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sum[i]), l)));
        }
    }
};
// o: a lane's sums, N to each of B blocks, fours of them being neighbours: element_of(four) is the first's element,
// index_of(element) the other way round (-1: not this lane's). below: the values that all rows see; each(visit) calls
// visit(key) for the keys that some rows do not: each lane looks at its row's own elements there.
template <int DT, int DP, int B, int N, typename V, typename P, typename S, typename T, typename I>
__device__ __forceinline__ void settle(V (&o)[B], NonfiniteSum<DT> & below, int sees, int D, P row_of, S each, T element_of, I index_of) {
    constexpr uint32_t E = DT == F16 ? 0x7C00u : 0x7F80u;
    uint32_t lost[(B * N + 31) / 32] = {}; // a bit for each sum that is NaN
#pragma unroll
    for (int j = 0; j < B * N; ++j) {
        const float x = o[j / N][j % N];
        lost[j / 32] |= x != x ? 1u << (j % 32) : 0;
        o[j / N][j % N] = x != x ? 0.0f : x;
    }
    below.template give<DP>([&](int e, float x) {
        const int at = index_of(e);
        uint32_t word = lost[0];
#pragma unroll
        for (int w = 1; w < (B * N + 31) / 32; ++w) word = at >> 5 == w ? lost[w] : word;
        const int mine = at >= 0 && (word >> (at & 31) & 1) ? at : -1;
#pragma unroll
        for (int j = 0; j < B * N; ++j) o[j / N][j % N] += mine == j ? x : 0.0f;
    });
    each([&](int key) {
        const uint8_t * row = row_of(key);
#pragma unroll
        for (uint32_t & w : lost) asm volatile("" : "+v"(w)); // (else a mask for each bit is kept over the loop)
#pragma unroll
        for (int f = 0; f < B * N / 4; ++f) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            u32x2 v = {0, 0};
            if (key < sees && element_of(f) < D) v = *reinterpret_cast<const u32x2 *>(row + 2 * element_of(f));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = 4 * f + i;
                const uint32_t h = v[i / 2] >> (16 * (i & 1)) & 0xFFFFu;
                o[j / N][j % N] += (h & E) == E && (lost[j / 32] >> (j % 32) & 1) ? nonfinite<DT>(h) : 0.0f;
            }
        }
    });
#pragma unroll
    for (int j = 0; j < B * N; ++j) {
        const float x = o[j / N][j % N];
        o[j / N][j % N] = (lost[j / 32] >> (j % 32) & 1) && x == 0.0f ? NAN : x;
    }
}

// agent-scope accesses: written through, and read past, the XCDs' L2s
__device__ __forceinline__ void put2(float * p, float a, float b) {
    const uint64_t v = (uint64_t) __float_as_uint(a) | (uint64_t) __float_as_uint(b) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float * p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t) v), __uint_as_float((uint32_t) (v >> 32)));
}

// The pieces of some rows' keys meet in memory: every piece's work-group has written its rows' sums
// with put2. True in the work-group that arrives last. Its counterpart of a release is that each wave's stores, at agent
// scope, are acknowledged before the work-group's arrival is counted; of an acquire, that the last to
// count reads with get2. The count is left at zero.
__device__ __forceinline__ bool last_to_arrive(uint32_t * count, int pieces, uint32_t * said) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) *said = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (*said != (uint32_t) pieces - 1) return false;
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

hipError_t launch_attention_rows(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream);
hipError_t launch_attention_tiles(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream);

} // namespace sgk
