// ATTENTION_PROMPT, and ATTENTION_PAGED's requests with many new tokens (include/scrapgpu/hip_ops.h):
// tiles of 128 query rows (gfx950, wave64).
#include "attention.h"

#include <algorithm>
#include <cmath>
#include <cstdio>

namespace sgk {
namespace {

constexpr int BR = 128; // query rows of a tile: 32 for each of 4 waves
constexpr int BK = 64;  // keys of a step

template <int DT>
__device__ __forceinline__ f32x16 mma(const f16x8 & a, const f16x8 & b, const f32x16 & c) {
    if constexpr (DT == BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}


// Steps of a piece at least, and steps that the longest tile must lose for the cut to pay: the pieces'
// sums go through memory, which costs all about as much as 6 steps (prompts of 13 requests, 4500
// tokens, 14/2 heads of 64: 26.5 us whole, 28.5 in pieces that save 4 steps; one of 1000, 32/8 heads
// of 128: 32.3 whole, 29.3 in pieces that save 8)
constexpr int kMinSteps = 8, kJoinSteps = 6;

// a work-group's work: one tile of a request's rows, one piece of its keys
struct Work {
    int b, r0;         // request, first row
    int q0, nq;        // the request's first token and its count
    int kv;            // its keys
    int64_t k0;        // prompts: its first key
    int s0, s1;        // the steps of the piece
    int px;            // the piece, counted over all tiles
    int first, pieces; // the tile's first, and how many have steps (at least one)
};

// The `turn`-th of the pieces of all tiles of all requests, the last ones first, counted on the device
// from the requests' lengths, 64 at a time in each wave. `want` > 0: as many work-groups per key head
// as the CUs hold; where the longest tile gains by it, the tiles are cut into pieces of one length such
// that all together make at most about that many (never more than `want` over one for each tile: the
// `room` of the sums and the arrival counts, one less than the grid's); 0: each tile is one piece. False: past
// the last, as the w.px-th of w.pieces work-groups (w.q0: where the last request's tokens end), or (w.pieces 0) no piece (the grid's last work-groups, which
// so delay none: 64 tokens over 6000, 53.9 -> 38.9 us).
template <bool PAGED>
__device__ __forceinline__ bool find_work(const AttnLaunch & a, int turn, int want, int room, Work & w) {
    const int lane = threadIdx.x & 63;
    const auto load = [&](int b, int & q0, int & nq, int & kv, int & k0, int & tiles, int & steps) __attribute__((always_inline)) {
        q0 = nq = kv = k0 = 0;
        if (b < a.B) {
            const int2 r = range_of(a.q_start, b, a.T);
            q0 = r.x;
            nq = r.y - r.x;
            if constexpr (PAGED) {
                kv = min(max(a.k_at[b], 0), a.W << a.shift);
            } else {
                const int2 k = range_of(a.k_at, b, a.Tk);
                k0 = k.x;
                kv = k.y - k.x;
            }
        }
        tiles = (nq * a.G + BR - 1) / BR;
        steps = (kv + BK - 1) / BK;
    };
    int q0, nq, kv, k0, tiles, steps;
    load(lane, q0, nq, kv, k0, tiles, steps);
    int per = 1 << 30; // steps of a piece
    if (want > 0) {
        const auto all = [&](auto of, auto join) __attribute__((always_inline)) {
            float v = of(tiles, steps);
            for (int b0 = 64; b0 < a.B; b0 += 64) {
                int x, y, z, u, n, m;
                load(b0 + lane, x, y, z, u, n, m);
                v = join(v, of(n, m));
            }
            for (int d = 1; d < 64 && d < a.B; d <<= 1) v = join(v, __shfl_xor(v, d));
            return __builtin_amdgcn_readfirstlane((int) fminf(v, 1.0e9f));
        };
        const auto sum = [](float x, float y) { return x + y; };
        const int longest = all([](int n, int m) { return n > 0 ? (float) m : 0.0f; }, [](float x, float y) { return fmaxf(x, y); });
        if (longest > kMinSteps + kJoinSteps) {
            // (sums as f32: rounded up)
            const int total = all([](int n, int m) { return 1.0001f * (float) n * (float) m; }, sum);
            per = max(kMinSteps, total / want + 1);
            // a tile's last piece is shorter: longer ones until they fit
            for (int i = 0; i < 3; ++i) {
                const int n = all([&](int n, int m) { return 1.0001f * (float) (n * max(1, (m + per - 1) / per)); }, sum);
                if (n <= want) break;
                per = max(per + 1, (int) ((int64_t) per * n / want));
            }
            if (longest <= per + kJoinSteps) per = 1 << 30;
        }
    }
    int cut, n, sum; // a tile's pieces, the request's, the pieces of all requests up to it
    const auto count = [&](int b0) __attribute__((always_inline)) {
        cut = max(1, (steps + per - 1) / per);
        sum = n = tiles * cut;
        for (int d = 1; d < 64 && d < a.B - b0; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        return __builtin_amdgcn_readlane(sum, min(63, a.B - 1 - b0));
    };
    const auto count_all = [&]() __attribute__((always_inline)) {
        int pieces = count(0);
        for (int b0 = 64; b0 < a.B; b0 += 64) {
            load(b0 + lane, q0, nq, kv, k0, tiles, steps);
            pieces += count(b0);
        }
        return pieces;
    };
    int pieces = count_all();
    if (pieces > room) { // (only where starts cover tokens twice: no pieces, whose sums and counts had no place)
        per = 1 << 30;
        if (a.B > 64) load(lane, q0, nq, kv, k0, tiles, steps);
        pieces = count_all();
    }
    const int px = pieces - 1 - turn;
    w.px = px;
    if (px < 0) {
        w.q0 = __builtin_amdgcn_readlane(q0 + nq, (a.B - 1) & 63);
        w.px = turn - pieces;
        w.pieces = room + 1 - pieces;
        return false;
    }
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        int here = pieces;
        if (a.B > 64) {
            load(b0 + lane, q0, nq, kv, k0, tiles, steps);
            here = count(b0);
        }
        const uint64_t hit = __ballot(b0 + lane < a.B && base + sum > px);
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            w.b = b0 + l;
            w.q0 = __builtin_amdgcn_readlane(q0, l);
            w.nq = __builtin_amdgcn_readlane(nq, l);
            w.kv = __builtin_amdgcn_readlane(kv, l);
            w.k0 = __builtin_amdgcn_readlane(k0, l);
            const int c = __builtin_amdgcn_readlane(cut, l), first = base + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l);
            const int tile = c == 1 ? px - first : (px - first) / c, piece = px - first - tile * c;
            w.r0 = tile * BR;
            w.first = first + tile * c;
            // as far as the tile's last row sees, in pieces of equal length
            const int last = min(w.nq - 1, (w.r0 + BR - 1) / a.G);
            const int end = a.causal ? min(max(w.kv - w.nq + last + 1, 0), w.kv) : w.kv, steps_here = (end + BK - 1) / BK;
            const int len = c == 1 ? steps_here : max(1, (steps_here + c - 1) / c);
            w.pieces = c == 1 ? 1 : max(1, (steps_here + len - 1) / len);
            w.s0 = piece * len;
            w.s1 = min(steps_here, w.s0 + len);
            if (piece < w.pieces) return true;
            w.pieces = 0; // (the tile has fewer steps than pieces)
            return false;
        }
        base += here;
    }
    w.pieces = 0;
    return false;
}

// One tile of 128 rows x one piece of its keys. A wave owns 32 rows: Q as operands in registers,
// O^T (DP x 32) and the softmax's statistics too. The keys go by in steps of 64: K and V of the next
// step are on their way into one half of LDS (straight from memory) while the present one is worked
// on in the other.
//
// Bound: the matrix units, which are busy 48% of the time, and the softmax between the two products:
// 64 weights a lane and step. Two work-groups a CU (heads of 128; 3 of 64, 1 of 256) cover one
// another's softmax and waits. 8192 tokens of 32/8 heads of 128 in bf16: 546 to 577 us from card to card, 0.95 to 1.01 PFLOP/s, where a
// large library product of that type reaches 1.10; F32 results (2 or 3 terms) 0.63 and 0.51 PFLOP/s
// at 4096 tokens, heads of 256 0.63. Tiles of 256 rows in 8 waves gave 3% at 8192 tokens and lost 11%
// on packed prompts; a third step on its way through the weights, or no maximum at all, gave nothing.
//
// LDS: a row of DP elements is DP / 8 chunks of 16 bytes; row r's chunk c sits at chunk c ^ f(r), so
// that the 16 rows of a K operand's read (one chunk each), and the 4 rows x 64 bytes that 32 lanes of a
// transposing read of V take together, lie in different banks (f(r) = 2 (r & 7), right for 32 bytes
// each, cost 4096 tokens of 32/8 heads of 64 91 us for 86).
template <int DT, int DW, bool PAGED, bool OUT32>
__global__ __launch_bounds__(256, DW == 256 ? 1 : 2) void k_attention(AttnLaunch a, float * scratch, uint32_t * arrive, int want) {
    constexpr int NT = OUT32 ? kTerms<DT> : 1; // terms of a weight
    constexpr int DP = padded(DW);        // elements between rows in LDS
    constexpr int NC = DP / 8;            // chunks of a row
    constexpr int RB = 2 * DP;            // bytes of a row
    constexpr int RI = 64 / NC;           // rows that one load instruction of a wave moves
    constexpr int NI = BK / RI / 4;       // instructions of a wave for a step's K (and for its V)
    constexpr int HALF = 2 * BK * RB;     // one step's K and V
    constexpr int DB = DW / 32, KT = DW / 16;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;

    // heads next to each other in the grid (work-groups go round the XCDs: with 8 key heads each
    // XCD's L2 holds one head's keys), a sequence's last tiles, which see the most keys, first
    const int kvh = blockIdx.x % a.Hk, turn = blockIdx.x / a.Hk;
    Work t;
    if (__builtin_expect(!find_work<PAGED>(a, turn, want, (int) (gridDim.x / a.Hk) - 1, t), 0)) {
        if (t.pieces > 0) zero_rest(a, t.q0, kvh, t.px, t.pieces);
        return;
    }
    const int s0 = t.s0, s1 = t.s1;
    // this lane's row, and how many keys it sees
    const int row = t.r0 + 32 * wid + n, tok = row / a.G;
    const bool live = tok < t.nq;
    const int head = kvh * a.G + (row - tok * a.G);
    const int sees = !live ? 0 : a.causal ? min(max(t.kv - t.nq + tok + 1, 0), t.kv) : t.kv;
    // (the first row of the tile sees the fewest: steps below are seen whole by all)
    // (and the wave's last row the most of the wave's: steps from there on it only loads)
    const int wave_last = min(t.r0 + 32 * wid + 31, t.nq * a.G - 1) / a.G;
    const int wave_sees = t.r0 + 32 * wid >= t.nq * a.G ? 0 : a.causal ? min(max(t.kv - t.nq + wave_last + 1, 0), t.kv) : t.kv;
    const int sees_all = a.causal ? max(t.kv - t.nq + t.r0 / a.G + 1, 0) : t.kv;

    f16x8 q[KT];
    {
        const uint8_t * p = a.q + (int64_t) (t.q0 + min(tok, t.nq - 1)) * a.q_s2 + (live ? head : kvh * a.G) * a.q_s1;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u; // (the scale's sign goes into q, so that maxima of scores are maxima of weights)
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            // (past D: the row's last elements, made zero; no branch, so that all loads are in flight at once)
            const u32x4 v = *reinterpret_cast<const u32x4 *>(p + min(2 * (16 * i + 8 * h), 2 * a.D - 16)) ^ flip;
            q[i] = __builtin_bit_cast(f16x8, 16 * i + 8 * h < a.D ? v : u32x4{0, 0, 0, 0});
        }
    }
    const float c = weight_scale(a);

    if (a.D < DP) { // the chunks past D stay zero
        for (int i = threadIdx.x; i < 2 * HALF / 16; i += 256) reinterpret_cast<u32x4 *>(lds)[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }

    // Loads. A wave moves 16 rows of a step's K and V; instruction i rows i RI .. of them, lane l its
    // chunk l % NC of row l / NC, and which chunk of memory that is follows from the place's f(r). The
    // 16 rows lie in one page (pages have 16 places or more), so a load's address is one base for the
    // wave and an offset that only the step past the end changes: rows past the last key read the
    // last key (their weights are zero).
    const uint8_t *kb = a.k + kvh * a.k_s2, *vb = a.v + kvh * a.v_s2;
    const auto fk = [](int r) { return DP == 64 ? (r >> 1) & 7 : r & 15; };
    const auto fv = [](int r) { return DP == 64 ? 4 * ((r >> 1) & 1) + 2 * ((r >> 2) & 1) : 4 * (r & 3) + 2 * ((r >> 2) & 1); };
    const int lr = lane / NC, lc = lane % NC;
    uint32_t offk[NI], offv[NI];
    const auto offsets = [&](int last) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = i * RI + lr;
            offk[i] = (uint32_t) min(r, last) * (uint32_t) a.k_s1 + 16 * (lc ^ fk(r));
            offv[i] = (uint32_t) min(r, last) * (uint32_t) a.v_s1 + 16 * (lc ^ fv(r));
        }
    };
    offsets(15);
    // the page of the wave's rows of step s, a step ahead of its use
    const auto page_of = [&](int s) __attribute__((always_inline)) { return PAGED ? a.table[t.b * a.t_s1 + (min(s * BK + 16 * wid, t.kv - 1) >> a.shift)] : 0; };
    const auto fetch = [&](int s, int page, int half) __attribute__((always_inline)) {
        const int k0 = min(s * BK + 16 * wid, t.kv - 1);
        if (s * BK + BK > t.kv) offsets(t.kv - 1 - k0); // (the last step)
        const uint8_t *pk, *pv;
        if constexpr (PAGED) {
            const uint64_t p = (uint32_t) min(max(__builtin_amdgcn_readfirstlane(page), 0), a.n_pages - 1);
            const uint32_t at = (uint32_t) k0 & ((1u << a.shift) - 1);
            pk = kb + p * (uint32_t) a.k_s3 + (uint64_t) at * (uint32_t) a.k_s1;
            pv = vb + p * (uint32_t) a.v_s3 + (uint64_t) at * (uint32_t) a.v_s1;
        } else {
            pk = kb + (uint64_t) (t.k0 + k0) * a.k_s1;
            pv = vb + (uint64_t) (t.k0 + k0) * a.v_s1;
        }
        uint8_t * d = lds + half * HALF + wid * NI * 1024;
        if (a.D == DP) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                load_lds16(pk, offk[i], d + i * 1024);
                load_lds16(pv, offv[i], d + BK * RB + i * 1024);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = i * RI + lr;
                if (8 * (lc ^ fk(r)) < a.D) load_lds16(pk, offk[i], d + i * 1024);
                if (8 * (lc ^ fv(r)) < a.D) load_lds16(pv, offv[i], d + BK * RB + i * 1024);
            }
        }
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = kNoMax, l = 0.0f; // (l: this half-wave's share)

    const uint32_t ka = n * RB + 16 * (h ^ fk(n));
    const int vr = 4 * h + ((lane & 15) >> 2);
    const uint32_t va = BK * RB + vr * RB + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ fv(vr)) + 8 * (lane & 1);
    const auto vread = [&](int half, int kt, int d) __attribute__((always_inline)) {
        const uint8_t * at = lds + 16 * kt * RB + ((half * HALF + va) ^ (64 * d));
        const s16x4 x = read_column4(at), y = read_column4(at + 8 * RB);
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    // (see has_nonfinite; the waves share the step's values: each looks through its own loads)
    const auto clean = [&](int s, int half) __attribute__((always_inline)) {
        uint8_t * vs = lds + half * HALF + BK * RB;
        bool bad = false;
#pragma unroll 1
        for (int i = 0; i < NI; ++i) bad |= has_nonfinite<DT>(reinterpret_cast<const u32x4 *>(vs + (wid * NI + i) * 1024)[lane]);
        if (!__syncthreads_or(bad)) return;
#pragma unroll 1
        for (int i = 0; i < 4 * NI; ++i) {
            const u32x4 v = reinterpret_cast<const u32x4 *>(vs + i * 1024)[lane];
            const int r = i * RI + lr;
            each_nonfinite<DT>(v, r * DP + 8 * (lc ^ fv(r)), [&](int e, float x) {
                const int key = s * BK + e / DP, el = e % DP - 4 * h;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[d][j] += key < sees && el == 32 * d + 8 * (j >> 2) + (j & 3) ? x : 0.0f;
            });
        }
        __syncthreads();
#pragma unroll 1
        for (int i = 0; i < NI; ++i) {
            u32x4 * at = reinterpret_cast<u32x4 *>(vs + (wid * NI + i) * 1024) + lane;
            *at = only_finite<DT>(*at);
        }
        __syncthreads();
    };

    // One step: the scores S^T = K Q^T, their weights, O^T += V^T P^T
    const auto step = [&](int s, int half) __attribute__((always_inline)) {
        const bool masked = (s + 1) * BK > sees_all;
        f32x16 sc[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[b][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                const f16x8 k = *reinterpret_cast<const f16x8 *>(lds + 32 * b * RB + ((half * HALF + ka) ^ (32 * i)));
                sc[b] = mma<DT>(k, q[i], sc[b]);
            }
        }
        // lane (n, h), register i of block b: key 64 s + 32 b + 8 (i / 4) + 4 h + i % 4
        if (masked) {
            const int left = sees - s * BK - 4 * h;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[b][i] = 32 * b + 8 * (i >> 2) + (i & 3) < left ? sc[b][i] : -INFINITY;
        }
        // (the other work-group's products go first: 575 -> 559 us at 8192 tokens, 32/8 heads of 128)
        __builtin_amdgcn_s_setprio(0);
        float mx = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) mx = fmaxf(mx, sc[e >> 4][e & 15]);
        mx = max_halves(mx) * c;
        if (__any(mx > m + kLag)) {
            const float to = fmaxf(m, mx), f = decay(m, to);
            m = to;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
        }
        const float off = kLift<DT> - m;
        u32x4 w[NT][4];
        float total = 0.0f;
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[e >> 4][e & 15], c, off)), p1 = __builtin_amdgcn_exp2f(fmaf(sc[e >> 4][(e & 15) + 1], c, off));
            if constexpr (OUT32) {
                total += p0;
                total += p1;
                uint32_t term[NT];
                split<DT, NT>(p0, p1, term);
#pragma unroll
                for (int n = 0; n < NT; ++n) w[n][e >> 3][e / 2 & 3] = term[n];
            } else {
                w[0][e >> 3][e / 2 & 3] = round2<DT>(p0, p1, total);
            }
        }
        l += total;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const f16x8 v = vread(half, kt, d);
#pragma unroll
                for (int n = 0; n < NT; ++n) o[d] = mma<DT>(v, __builtin_bit_cast(f16x8, w[n][kt]), o[d]);
            }
    };

    if (s0 < s1) {
        fetch(s0, page_of(s0), 0);
        int page = page_of(min(s0 + 1, s1 - 1));
        for (int s = s0; s < s1; ++s) {
            const int half = (s - s0) & 1;
            // this step's K and V are in LDS, and no wave reads the other half any more
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (s + 1 < s1) {
                fetch(s + 1, page, half ^ 1);
                page = page_of(min(s + 2, s1 - 1));
            }
            if ((s + 1) * BK > sees_all) clean(s, half);
            if (s * BK < wave_sees) step(s, half);
        }
    }

    { // (a NaN among the sums: see settle)
        float any[4] = {0.0f, 0.0f, 0.0f, 0.0f}; // (two of them an instruction: a NaN spreads through the products)
#pragma unroll
        for (int j = 0; j < DB * 16; j += 2) any[j / 2 & 3] = fmaf(o[j / 16][j % 16], o[j / 16][j % 16 + 1], any[j / 2 & 3]);
        const float sum = (any[0] + any[1]) + (any[2] + any[3]);
        if (__builtin_expect(__any(sees > 0 && sum != sum), 0)) {
            const auto row_of = [&](int key) {
                if constexpr (!PAGED) return vb + (uint64_t) (t.k0 + key) * a.v_s1;
                const uint64_t page = (uint32_t) min(max(a.table[t.b * a.t_s1 + (key >> a.shift)], 0), a.n_pages - 1);
                return vb + page * a.v_s3 + (uint64_t) (key & ((1 << a.shift) - 1)) * a.v_s1;
            };
            const int from = s0 * BK, to = min(s1 * BK, t.kv), apart = max(from, min(to, sees_all));
            NonfiniteSum<DT> below;
            below.template take<DP>(from, apart, a.D, row_of);
            settle<DT, DP, DB, 16>(
                o, below, sees, a.D, row_of,
                [&](auto visit) {
#pragma unroll 1
                    for (int key = apart; key < to; ++key) visit(key);
                },
                [&](int four) { return 32 * (four >> 2) + 8 * (four & 3) + 4 * h; },
                [&](int e) {
                    const int at = e - 4 * h; // 32 block + 8 (i / 4) + i % 4
                    return at >= 0 && (at & 4) == 0 ? 16 * (at >> 5) + 4 * (at >> 3 & 3) + (at & 3) : -1;
                });
        }
    }

    l = sum_halves(l);
    if (t.pieces > 1) {
        // The pieces of the tile meet in memory: each writes its sums as its lanes hold them (512
        // consecutive bytes a store), the last to arrive adds all in order, for all its waves' rows.
        constexpr int ITEM = BR * (DP + 2);
        float * part = scratch + ((int64_t) t.first * a.Hk + kvh) * ITEM;
        const int64_t gap = (int64_t) a.Hk * ITEM;
        float * mine = part + (t.px - t.first) * gap;
        const bool some = t.r0 + 32 * wid < t.nq * a.G; // (waves without a row have nothing to say)
        if (some) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 8; ++e) put2(mine + (((wid * DB + d) * 8 + e) * 64 + lane) * 2, o[d][2 * e], o[d][2 * e + 1]);
            if (h == 0) put2(mine + BR * DP + (32 * wid + n) * 2, m, l);
        }
        __syncthreads(); // (LDS: the last step's reads are over)
        if (!last_to_arrive(arrive + (int64_t) t.first * a.Hk + kvh, t.pieces, reinterpret_cast<uint32_t *>(lds))) return;
        if (!some) return;
        m = kNoMax;
        l = 0.0f;
#pragma unroll 1
        for (int p = 0; p < t.pieces; ++p) m = fmaxf(m, get2(part + p * gap + BR * DP + (32 * wid + n) * 2).x);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
#pragma unroll 1
        for (int p = 0; p < t.pieces; ++p) {
            const float * from = part + p * gap;
            const float2 st = get2(from + BR * DP + (32 * wid + n) * 2);
            const float f = decay(st.x, m);
            l = fmaf(st.y, f, l);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float2 v = get2(from + (((wid * DB + d) * 8 + e) * 64 + lane) * 2);
                    o[d][2 * e] = fmaf(v.x, f, o[d][2 * e]);
                    o[d][2 * e + 1] = fmaf(v.y, f, o[d][2 * e + 1]);
                }
        }
    }
    // (no key: zeros; keys whose scores are all -Inf: 0 / 0)
    const float inv = sees == 0 ? 0.0f : 1.0f / l;
    if (live) {
        uint8_t * out = a.o + (int64_t) (t.q0 + tok) * a.o_s2 + head * a.o_s1;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = 32 * d + 8 * j + 4 * h;
                if (at < a.D) store4<DT, OUT32>(out, at, o[d][4 * j] * inv, o[d][4 * j + 1] * inv, o[d][4 * j + 2] * inv, o[d][4 * j + 3] * inv);
            }
    }
}

template <int DT, int DW, bool PAGED, bool OUT32>
hipError_t go(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    const size_t lds = (size_t) 4 * BK * 2 * padded(DW);
    const hipError_t e = allow_lds((void *) k_attention<DT, DW, PAGED, OUT32>, lds);
    if (e != hipSuccess) return e;
    last_form().grid = (uint64_t) attention_groups(a, s);
    k_attention<DT, DW, PAGED, OUT32><<<dim3((unsigned) last_form().grid), dim3(256), lds, stream>>>(a, reinterpret_cast<float *>(scratch), arrive, s.want);
    return hipGetLastError();
}

template <int DT, bool PAGED, bool OUT32>
hipError_t by_dim(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    if (a.D <= 64) return go<DT, 64, PAGED, OUT32>(a, s, scratch, arrive, stream);
    if (a.D <= 96) return go<DT, 96, PAGED, OUT32>(a, s, scratch, arrive, stream);
    if (a.D <= 128) return go<DT, 128, PAGED, OUT32>(a, s, scratch, arrive, stream);
    return go<DT, 256, PAGED, OUT32>(a, s, scratch, arrive, stream);
}

template <int DT>
hipError_t by_form(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    const bool o32 = a.out_type == F32;
    if (a.table) return o32 ? by_dim<DT, true, true>(a, s, scratch, arrive, stream) : by_dim<DT, true, false>(a, s, scratch, arrive, stream);
    return o32 ? by_dim<DT, false, true>(a, s, scratch, arrive, stream) : by_dim<DT, false, false>(a, s, scratch, arrive, stream);
}

} // namespace

hipError_t launch_attention_tiles(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    return a.dtype == F16 ? by_form<F16>(a, s, scratch, arrive, stream) : by_form<BF16>(a, s, scratch, arrive, stream);
}

AttnShape attention_shape(const AttnLaunch & a, int cu_count, bool lean) {
    AttnShape s{};
    const int DP = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
    const int64_t rows = (int64_t) a.T * a.G, longest = (int64_t) a.max_query * a.G;
    const int64_t room = (int64_t) (lean ? 32 : 96) << 20; // bytes of partial sums
    // Single tokens, or a few (64 rows fit the registers, 16 of 256 elements), over the cache: the
    // kernel for few rows. No more tokens than requests: the same, whatever max_query says.
    const int most_nb = DP == 256 ? 1 : 4;
    s.few = a.paged && (longest <= 16 * most_nb || a.T <= a.B) && (int64_t) a.B * a.Hk <= kArriveMax;
    if (s.few) {
        s.nb = longest <= 16 ? 1 : std::min(longest <= 32 ? 2 : 4, most_nb);
        const int64_t piece = (int64_t) 16 * s.nb * (DP + 2) * 4 * a.Hk;
        const int64_t fit = room / piece - a.B;
        // As many work-groups as the CUs hold at once, two each or one (8 requests of 64 rows of 96 over up to
        // 20000, 128/2 heads: 58.9 us with one for each CU, 85.7 with two); where the requests alone make two
        // for each CU, four, which even out unequal histories (64 of up to 8000 keys, 8 heads: 147 -> 138 us,
        // 64 of up to 6000 of 256 elements 247 -> 232; but 16 of up to 8000 43.5 -> 45.4, 2 of 131071 99.5 -> 109).
        const int64_t many = (int64_t) ((int64_t) a.B * a.Hk >= 2 * cu_count ? 4 : std::min(2, resident(DP, s.nb))) * cu_count / a.Hk;
        s.want = (int) std::max<int64_t>(0, std::min(std::max<int64_t>(many, 1), fit));
        s.scratch = s.want > 0 ? (size_t) ((s.want + a.B) * piece) : 0; // (no room: requests whole)
        // work-groups without a piece: one, or what 32 KiB of zeros each ask for
        const int64_t unused = std::max<int64_t>(0, a.T - (int64_t) a.B * a.max_query), zeros = unused * a.G * a.D * (a.out_type == F32 ? 4 : 2);
        s.idle = (int) std::max<int64_t>(1, std::min<int64_t>(zeros >> 15, 2 * cu_count / a.Hk));
        return s;
    }
    // Tiles of all requests at most; fewer than the work-groups that the CUs hold at once: the keys may
    // be cut into pieces, within the scratch and the arrival counts, which the device decides from the
    // lengths (512 tokens over 6000 beside 15 single ones, 32/8 heads of 128: 139 -> 102 us; twice 512
    // over 20000, 16/8 heads of 256: 930 -> 374)
    s.tiles = (int) (rows / BR + std::min<int64_t>(a.B, rows));
    const int64_t slots = (int64_t) cu_count * (DP == 64 ? 3 : DP == 128 ? 2 : 1), item = (int64_t) BR * (DP + 2) * 4;
    if ((int64_t) s.tiles * a.Hk < slots) {
        const int64_t fit = std::min<int64_t>(room / item, kArriveMax) / a.Hk - s.tiles;
        s.want = (int) std::max<int64_t>(0, std::min<int64_t>(slots / a.Hk, fit));
        s.scratch = s.want > 0 ? (size_t) ((s.tiles + s.want) * a.Hk * item) : 0;
    }
    return s;
}

int64_t attention_groups(const AttnLaunch & a, const AttnShape & s) {
    return (s.few ? (int64_t) s.want + a.B + s.idle : (int64_t) s.tiles + s.want + 1) * a.Hk;
}

hipError_t launch_attention(const AttnLaunch & a, uint8_t * scratch, uint32_t * arrive, int cu_count, bool lean, hipStream_t stream) {
    const AttnShape s = attention_shape(a, cu_count, lean);
    if (s.few) std::snprintf(last_form().form, sizeof(last_form().form), "attention rows nb=%d want=%d", s.nb, s.want);
    else std::snprintf(last_form().form, sizeof(last_form().form), "attention tiles want=%d", s.want);
    return s.few ? launch_attention_rows(a, s, scratch, arrive, stream) : launch_attention_tiles(a, s, scratch, arrive, stream);
}

} // namespace sgk
