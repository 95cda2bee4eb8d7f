// ATTENTION_PAGED's requests with few new tokens (include/scrapgpu/hip_ops.h): single tokens of
// generation, or a handful of them, over the paged cache (gfx950, wave64).
//
// Bound: the cache's bytes. All rows of a request that share a key head (new tokens x G heads) are
// one block of 16 rows, or 2 or 4 of them, so the keys and values of a head are read once. 64 tokens
// over histories of up to 8000, 32/8 heads of 128: 724 MB in 135 us, 5.4 TB/s; two over 131071: 572 MB
// in 97 us, 5.9 TB/s (reads alone reach 6.45); one over 900: 9.2 us, latency.
//
// Split. The keys of all requests are cut into pieces of one length, chosen on the device from the
// requests' lengths so that the pieces of all requests together are about as many as the CUs hold
// work-groups: a batch of unequal histories is then as balanced as one of equal ones, whatever the
// table's width. A work-group is one piece of one key head; its 4 waves take steps of 32 keys in
// turn, each with a softmax of its own, and meet once, at the end, in LDS. The pieces of a request
// meet in memory, where the last to arrive adds them in order.
//
// A wave's step. K goes straight into registers as the first product's operand (a lane reads 16
// bytes of one key; the four lane parts of a key cover 64 bytes); V goes straight into LDS and comes
// out through transposing reads. The next step's K and V are asked for as soon as the first product
// has read the present K's registers (one copy of K, two places for V), and are on their way through
// the weights and the second product. Nothing is shared between waves, so there is no barrier in the
// loop.
#include "attention.h"

#include <algorithm>
#include <cstdio>

namespace sgk {
namespace {

constexpr int SK = 32;    // keys of a wave's step
constexpr int kWaves = 4;

template <int DT>
__device__ __forceinline__ f32x4 mma16(const f16x8 & a, const f16x8 & b, const f32x4 & c) {
    if constexpr (DT == BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// over the four lanes of a row (lane % 16 the same)
__device__ __forceinline__ float2 both_quarters(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t lo = r[0], hi = r[1];
    return make_float2(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float max_row(float v) {
    const float2 r = both_quarters(max_halves(v));
    return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float sum_row(float v) {
    const float2 r = both_quarters(sum_halves(v));
    return r.x + r.y;
}

struct Piece {
    int b, q0, nq, kv; // the request, its new tokens, its keys
    int s0, s1;        // its steps in this piece
    int first, count;  // the request's pieces, counted over all requests
};

// Piece `px` of the pieces of all requests. `want`: pieces wished for in all; 0: one a request. A
// request of more rows than `limit` (more new tokens than the caller said) is one piece. False: past the
// last, as the p.first-th of p.count work-groups (p.q0: where the last request's tokens end).
__device__ __forceinline__ bool find_piece(const AttnLaunch & a, int px, int want, int limit, Piece & p) {
    const int lane = threadIdx.x & 63;
    const auto load = [&](int b, int & q0, int & nq, int & kv, int & steps) {
        q0 = nq = kv = steps = 0;
        if (b >= a.B) return;
        const int2 r = range_of(a.q_start, b, a.T);
        q0 = r.x;
        nq = r.y - r.x;
        kv = min(max(a.k_at[b], 0), a.W << a.shift);
        steps = nq == 0 ? 0 : (kv + SK - 1) / SK;
    };
    int q0, nq, kv, steps;
    load(lane, q0, nq, kv, steps);
    float sum_all = (float) steps; // (as f32: rounded up below)
    for (int b0 = 64; b0 < a.B; b0 += 64) {
        int x, y, z, n;
        load(b0 + lane, x, y, z, n);
        sum_all += (float) n;
    }
    for (int d = 1; d < 64 && d < a.B; d <<= 1) sum_all += __shfl_xor(sum_all, d);
    // (steps of a piece, so many that there are at most `want` pieces and one more a request, which the grid, the
    // sums and the arrival counts hold, however long all together are; the sum is the same in every lane: said
    // so, the pieces' bounds and all that follows stay scalar)
    const float all = sum_all * 1.0001f;
    const int share = want == 0 ? 1 << 30 : all < 1.0e9f ? ((int) all + 1) / want : (int) fminf(all / (float) want, 1.0e9f) + 1;
    const int per = __builtin_amdgcn_readfirstlane(max(kWaves, (share + kWaves) / kWaves * kWaves));
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (b0 > 0) load(b0 + lane, q0, nq, kv, steps);
        // (the join reads every piece: a long request's pieces are longer, such that a wave's time for
        // one piece grows as fast as the join's shrinks. 8000 keys, 8 heads: 62 pieces 19.7 us, 31 16.6,
        // 21 17.5; 30000 keys, 1 head: 234 pieces 25.7, 59 20.2)
        const int least = max(per, kWaves * (int) (sqrtf((float) steps * (1.0f / (14 * kWaves))) + 0.5f));
        const int n = nq == 0 ? 0 : nq * a.G > limit ? 1 : max(1, (steps + least - 1) / least);
        int sum = n;
        for (int d = 1; d < 64 && d < a.B - b0; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const uint64_t hit = __ballot(b0 + lane < a.B && base + sum > px);
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            p.b = b0 + l;
            p.q0 = __builtin_amdgcn_readlane(q0, l);
            p.nq = __builtin_amdgcn_readlane(nq, l);
            p.kv = __builtin_amdgcn_readlane(kv, l);
            p.count = __builtin_amdgcn_readlane(n, l);
            p.first = base + __builtin_amdgcn_readlane(sum, l) - p.count;
            const int all = __builtin_amdgcn_readlane(steps, l), at = px - p.first;
            // (of equal length, whole rounds of the waves; the last may be empty)
            const int len = p.count == 1 ? all : ((all + p.count - 1) / p.count + kWaves - 1) / kWaves * kWaves;
            p.s0 = min(all, at * len);
            p.s1 = min(all, p.s0 + len);
            return true;
        }
        base += __builtin_amdgcn_readlane(sum, min(63, a.B - 1 - b0));
    }
    p.q0 = __builtin_amdgcn_readlane(q0 + nq, (a.B - 1) & 63);
    p.first = px - base;
    p.count = (int) (gridDim.x / a.Hk) - base;
    return false;
}

// Adds the sums of `pieces` pieces (DP floats, the maximum and the total, DP + 2 a row; piece p's at
// part + p * gap) of a request's `rows` rows and stores the results; `seen`: the keys that the first
// new token sees. A thread owns 4 elements of a row; where that leaves threads over, they take every
// so-many-th piece each, 8 pieces' loads at a time, and meet in LDS (`meet`: 6 floats a thread). The
// order of the additions is fixed.
template <int DT, int DP>
__device__ __forceinline__ void join_pieces(const AttnLaunch & a, const float * part, int64_t gap, int pieces, int rows, int q0, int kvh, int seen, float * meet) {
    constexpr int T = 64 * kWaves, Q = DP / 4;
    const int items = rows * Q, share = items <= T / 2 ? T / items : 1; // threads for an item
    for (int i0 = 0; i0 < items; i0 += T / share) {
        const int i = i0 + (int) threadIdx.x % (T / share), turn = threadIdx.x / (T / share);
        const bool mine = i < items && turn < share;
        const int r = i / Q, d = 4 * (i % Q);
        float top = kNoMax, total = 0.0f;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        const auto add = [&](float m, float l, f32x4 v) __attribute__((always_inline)) {
            const float f = decay(m, top);
            total = fmaf(l, f, total);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(v[e], f, x[e]);
        };
        const auto raise = [&](float to) __attribute__((always_inline)) {
            const float f = decay(top, to);
            top = to;
            total *= f;
            x *= f;
        };
        for (int g = turn; mine && g < pieces; g += 8 * share) {
            float2 st[8], u[8], v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float * at = part + min(g + k * share, pieces - 1) * gap + r * (DP + 2);
                st[k] = get2(at + DP);
                u[k] = get2(at + d);
                v[k] = get2(at + d + 2);
            }
            float to = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) to = fmaxf(to, st[k].x);
            raise(to);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (g + k * share < pieces) add(st[k].x, st[k].y, f32x4{u[k].x, u[k].y, v[k].x, v[k].y});
        }
        if (share > 1) {
            float * own = meet + threadIdx.x * 6;
            own[0] = top;
            own[1] = total;
#pragma unroll
            for (int e = 0; e < 4; ++e) own[2 + e] = x[e];
            __syncthreads();
            for (int k = 1; turn == 0 && k < share; ++k) {
                const float * o = own + k * (T / share) * 6;
                raise(fmaxf(top, o[0]));
                add(o[0], o[1], f32x4{o[2], o[3], o[4], o[5]});
            }
        }
        if (!mine || turn != 0 || d >= a.D) continue;
        const int tok = r / a.G;
        const float inv = (a.causal ? seen + tok : seen) <= 0 ? 0.0f : 1.0f / total;
        uint8_t * y = a.o + (int64_t) (q0 + tok) * a.o_s2 + (int64_t) (kvh * a.G + r - tok * a.G) * a.o_s1;
        if (a.out_type == F32) store4<DT, true>(y, d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        else store4<DT, false>(y, d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
}

template <int DT, int DW, int NB, int NT>
__global__ __launch_bounds__(64 * kWaves, resident(padded(DW), NB)) void k_attention_rows(AttnLaunch a, float * scratch, uint32_t * arrive, int want) {
    constexpr int DP = padded(DW);     // elements between rows in LDS and memory
    constexpr int NC = DP / 8;         // 16-byte chunks of a row
    constexpr int RB = 2 * DP;         // bytes of a row
    constexpr int RI = 64 / NC;        // rows of V that one load instruction moves
    constexpr int NV = SK / RI;        // load instructions of a step's V
    constexpr int NK = DW / 32;        // 16 keys x 32 elements each
    constexpr int DB = DW / 16;
    constexpr int TILE = SK * RB;      // one step's V
    constexpr int ROWS = 16 * NB;
    constexpr int OS = DP + 4;         // floats between rows of the waves' sums in LDS
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, part = lane >> 4;
    const int kvh = blockIdx.x % a.Hk, px = blockIdx.x / a.Hk;
    Piece p;
    if (__builtin_expect(!find_piece(a, px, want, ROWS, p), 0)) {
        zero_rest(a, p.q0, kvh, p.first, p.count);
        return;
    }
    const int rows = p.nq * a.G;
    const float c = weight_scale(a);
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
    const uint8_t *kb = a.k + kvh * a.k_s2, *vb = a.v + kvh * a.v_s2;
    uint8_t * mine = lds + wid * 2 * TILE; // two steps' V
    const auto fv = [](int r) { return DP == 64 ? 2 * ((r >> 1) & 3) : 2 * (r & 7); };
    // V operand: see k_attention; here the 16-lane group `part` takes rows 4 part .. + 3, then those 16
    // on. Elements 16 d on of a row are chunks 2 d and 2 d + 1, so d flips bits of the address.
    const int vr = 4 * part + (n >> 2);
    const uint32_t va = wid * 2 * TILE + vr * RB + 16 * (((n & 3) >> 1) ^ fv(vr)) + 8 * (n & 1);

    for (int r0 = 0; r0 < rows; r0 += ROWS) {
        f16x8 q[NB][NK];
        int sees[NB];
        int least = 0x7FFFFFFF; // keys that every row sees
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int row = r0 + 16 * b + n, tok = min(row / a.G, p.nq - 1), head = min(row - tok * a.G, a.G - 1);
            sees[b] = row >= rows ? 0 : a.causal ? min(max(p.kv - p.nq + tok + 1, 0), p.kv) : p.kv;
            const uint8_t * src = a.q + (int64_t) (p.q0 + tok) * a.q_s2 + (int64_t) (kvh * a.G + head) * a.q_s1;
#pragma unroll
            for (int t = 0; t < NK; ++t) {
                const u32x4 v = *reinterpret_cast<const u32x4 *>(src + min(2 * (32 * t + 8 * part), 2 * a.D - 16)) ^ flip;
                q[b][t] = __builtin_bit_cast(f16x8, 32 * t + 8 * part < a.D ? v : u32x4{0, 0, 0, 0});
            }
        }
        least = a.causal ? max(p.kv - p.nq + r0 / a.G + 1, 0) : p.kv;

        f32x4 o[NB][DB];
        float m[NB], l[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = kNoMax;
            l[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[b][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // A step's loads. Its two blocks of 16 keys lie in a page each (pages have 16 places or more):
        // a base for the wave and an offset a lane (V: one for each of the 8 / RI instructions after
        // which the places' permutation repeats). In the step past the end, keys past the last read
        // the last one. Chunks past D read the row's last (their elements of K are made zero before
        // use, their columns of O are never stored).
        constexpr int NP = RI >= 8 ? 1 : 8 / RI;
        const uint32_t offk = (uint32_t) n * (uint32_t) a.k_s1 + 16 * part;
        uint32_t offv[NP];
        const auto chunk_v = [&](int r) __attribute__((always_inline)) { return (uint32_t) min(16 * ((lane % NC) ^ fv(r)), 2 * a.D - 16); };
#pragma unroll
        for (int i = 0; i < NP; ++i) offv[i] = (uint32_t) (i * RI + lane / NC) * (uint32_t) a.v_s1 + chunk_v(i * RI + lane / NC);
        // the table's entries for the two blocks of step s (past the end: for the last key), a step ahead
        // of their use
        int entry[2];
        const auto look_up = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) entry[j] = a.table[p.b * a.t_s1 + (min(s * SK + 16 * j, p.kv - 1) >> a.shift)];
        };
        f16x8 k[2][NK];
        // V first: where K is there, V is
        const auto fetch = [&](int s, uint32_t half) __attribute__((always_inline)) {
            const bool inside = s * SK + SK <= p.kv;
            const uint8_t *pk[2], *pv[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint64_t page = (uint32_t) min(max(__builtin_amdgcn_readfirstlane(entry[j]), 0), a.n_pages - 1);
                const uint32_t at = (uint32_t) min(s * SK + 16 * j, p.kv - 1) & ((1u << a.shift) - 1);
                pk[j] = kb + page * (uint32_t) a.k_s3 + (uint64_t) at * (uint32_t) a.k_s1;
                pv[j] = vb + page * (uint32_t) a.v_s3 + (uint64_t) at * (uint32_t) a.v_s1;
            }
            look_up(s + kWaves);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = i * RI / 16;
                const uint8_t * src = pv[j] + (inside ? i * RI % 16 / 8 * 8 : 0) * (uint64_t) (uint32_t) a.v_s1;
                uint32_t off = offv[i % NP];
                if (!inside) {
                    const int r = i * RI + lane / NC;
                    off = (uint32_t) max(min(r % 16, p.kv - 1 - s * SK - 16 * j), 0) * (uint32_t) a.v_s1 + chunk_v(r);
                }
                load_lds16_once(src, off, mine + half + i * 1024);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (inside && a.D == DW) {
#pragma unroll
                    for (int t = 0; t < NK; ++t) k[j][t] = __builtin_bit_cast(f16x8, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(pk[j] + offk + 64 * t)));
                } else {
                    const uint32_t row = (uint32_t) max(min(n, p.kv - 1 - s * SK - 16 * j), 0) * (uint32_t) a.k_s1;
#pragma unroll
                    for (int t = 0; t < NK; ++t)
                        k[j][t] = __builtin_bit_cast(f16x8, __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(pk[j] + row + min(64 * t + 16 * part, 2 * a.D - 16))));
                }
            }
        };
        const auto vread = [&](uint32_t half, int d) __attribute__((always_inline)) {
            const uint8_t * at = lds + half + (va ^ (32 * d));
            const s16x4 x = read_column4(at), y = read_column4(at + 16 * RB);
            return __builtin_bit_cast(f16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        int s = p.s0 + wid;
        if (s < p.s1) {
            look_up(s);
            fetch(s, 0);
        }
        uint32_t half = 0;
        while (s < p.s1) {
            const int next = s + kWaves;
            const bool more = next < p.s1;
            const bool masked = (s + 1) * SK > least; // (rows past the last do not count: nobody reads what becomes of them)
            if (a.D < DW) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int t = 0; t < NK; ++t)
                        if (32 * t + 8 * part >= a.D) k[j][t] = f16x8{0, 0, 0, 0, 0, 0, 0, 0};
            }
            f32x4 sc[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    sc[b][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int t = 0; t < NK; ++t) sc[b][j] = mma16<DT>(k[j][t], q[b][t], sc[b][j]);
                }
            // (K's last load has been waited for above: everything before it is there, so this step's V)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (more) fetch(next, half ^ TILE);
            u32x4 w[NB][NT];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // lane (n, part), register i of block j: key 32 s + 16 j + 4 part + i
                const int left = sees[b] - s * SK - 4 * part;
                float x[8], mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = 16 * (i >> 2) + (i & 3) < left ? sc[b][i >> 2][i & 3] : -INFINITY;
                    mx = fmaxf(mx, x[i]);
                }
                mx = max_row(mx) * c;
                if (__any(mx > m[b] + kLag)) {
                    const float to = fmaxf(m[b], mx), f = decay(m[b], to);
                    m[b] = to;
                    l[b] *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[b][d] *= f;
                }
                const float off = kLift<DT> - m[b];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], c, off));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t term[NT];
                    l[b] += x[2 * i] + x[2 * i + 1];
                    split<DT, NT>(x[2 * i], x[2 * i + 1], term);
#pragma unroll
                    for (int n = 0; n < NT; ++n) w[b][n][i] = term[n];
                }
            }
            if (masked) {
                // (see has_nonfinite; the step's values are this wave's alone)
#pragma unroll 1
                for (int i = 0; i < NV; ++i) {
                    u32x4 * place = reinterpret_cast<u32x4 *>(mine + half + i * 1024) + lane;
                    const u32x4 v = *place;
                    if (!__any(has_nonfinite<DT>(v))) continue;
                    const int r = i * RI + lane / NC;
                    each_nonfinite<DT>(v, r * DP + 8 * ((lane % NC) ^ fv(r)), [&](int e, float x) {
                        const int key = s * SK + e / DP, el = e % DP - 4 * part;
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int d = 0; d < DB; ++d)
#pragma unroll
                                for (int j = 0; j < 4; ++j) o[b][d][j] += key < sees[b] && el == 16 * d + j ? x : 0.0f;
                    });
                    *place = only_finite<DT>(v);
                }
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const f16x8 v = vread(half, d);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n) o[b][d] = mma16<DT>(v, __builtin_bit_cast(f16x8, w[b][n]), o[b][d]);
            }
            half ^= TILE;
            s = next;
        }

        // (a NaN among the sums: see settle)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float any[2] = {0.0f, 0.0f}; // (two of them an instruction: a NaN spreads through the products)
#pragma unroll
            for (int j = 0; j < DB * 4; j += 2) any[j / 2 & 1] = fmaf(o[b][j / 4][j % 4], o[b][j / 4][j % 4 + 1], any[j / 2 & 1]);
            const float sum = any[0] + any[1];
            if (__builtin_expect(!__any(sees[b] > 0 && sum != sum), 1)) continue;
            const auto row_of = [&](int key) {
                const uint64_t page = (uint32_t) min(max(a.table[p.b * a.t_s1 + (key >> a.shift)], 0), a.n_pages - 1);
                return vb + page * a.v_s3 + (uint64_t) (key & ((1 << a.shift) - 1)) * a.v_s1;
            };
            NonfiniteSum<DT> below;
#pragma unroll 1
            for (int at = p.s0 + wid; at < p.s1; at += kWaves) below.template take<DP>(at * SK, min(min(at * SK + SK, p.kv), least), a.D, row_of);
            settle<DT, DP, DB, 4>(
                o[b], below, sees[b], a.D, row_of,
                [&](auto visit) {
#pragma unroll 1
                    for (int at = p.s0 + wid; at < p.s1; at += kWaves)
#pragma unroll 1
                        for (int key = max(at * SK, least); key < min(at * SK + SK, p.kv); ++key) visit(key);
                },
                [&](int four) { return 16 * four + 4 * part; },
                [&](int e) {
                    const int at = e - 4 * part; // 16 block + i
                    return at >= 0 && (at & 12) == 0 ? 4 * (at >> 4) + (at & 3) : -1;
                });
        }

        // the waves' sums meet in LDS, 16 rows at a time (the lane's number anew: addresses from here on
        // are formed here, and hold no registers through the loop above)
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        float * sums = reinterpret_cast<float *>(lds);                    // [wave][row][OS]
        float * stat = sums + kWaves * 16 * OS;                           // [wave][row][m, l]
        const bool joined = p.count > 1;
        float * out_part = scratch + ((int64_t) px * a.Hk + kvh) * (ROWS * (DP + 2));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (r0 + 16 * b >= rows) break;
            __syncthreads();
            const float lt = sum_row(l[b]);
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4 *>(sums + (wid * 16 + (tid & 15)) * OS + 16 * d + 4 * (tid >> 4 & 3)) = o[b][d];
            if ((tid & 48) == 0) {
                stat[(wid * 16 + (tid & 15)) * 2] = m[b];
                stat[(wid * 16 + (tid & 15)) * 2 + 1] = lt;
            }
            __syncthreads();
            const int r = tid >> 4, row = r0 + 16 * b + r;
            if (row < rows) {
                float top = kNoMax, total = 0.0f, f[kWaves];
#pragma unroll
                for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stat[(w * 16 + r) * 2]);
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    f[w] = decay(stat[(w * 16 + r) * 2], top);
                    total = fmaf(stat[(w * 16 + r) * 2 + 1], f[w], total);
                }
                const int tok = row / a.G;
                const int see = a.causal ? p.kv - p.nq + tok + 1 : p.kv;
                const float inv = see <= 0 || p.kv == 0 ? 0.0f : 1.0f / total;
                uint8_t * y = a.o + (int64_t) (p.q0 + tok) * a.o_s2 + (int64_t) (kvh * a.G + row - tok * a.G) * a.o_s1;
#pragma unroll
                for (int e = 0; e < DP / 64; ++e) {
                    const int d = 64 * e + 4 * (tid & 15);
                    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) v += *reinterpret_cast<const f32x4 *>(sums + (w * 16 + r) * OS + d) * f[w];
                    if (joined) {
                        float * at = out_part + (16 * b + r) * (DP + 2) + d;
                        put2(at, v[0], v[1]);
                        put2(at + 2, v[2], v[3]);
                    } else if (d < a.D) {
                        if (a.out_type == F32) store4<DT, true>(y, d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                        else store4<DT, false>(y, d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                    }
                }
                if (joined && (tid & 15) == 0) put2(out_part + (16 * b + r) * (DP + 2) + DP, top, total);
            }
        }
        if (!joined) {
            __syncthreads(); // (the next rows' V goes where the sums are)
            continue;
        }
        // (a request cut into pieces has at most ROWS rows: r0 is 0)
        if (last_to_arrive(arrive + p.b * a.Hk + kvh, p.count, reinterpret_cast<uint32_t *>(stat + kWaves * 16 * 2)))
            join_pieces<DT, DP>(a, scratch + ((int64_t) p.first * a.Hk + kvh) * (ROWS * (DP + 2)), (int64_t) a.Hk * (ROWS * (DP + 2)), p.count, rows, p.q0, kvh,
                                a.causal ? p.kv - p.nq + 1 : p.kv, sums);
        return;
    }
}

template <int DT, int DW, int NB, int NT>
hipError_t go(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    constexpr int DP = padded(DW);
    const size_t sums = (size_t) kWaves * 16 * (DP + 4) * 4 + kWaves * 16 * 8 + 16;
    const size_t lds = std::max((size_t) kWaves * 2 * SK * 2 * DP, sums);
    const hipError_t e = allow_lds((void *) k_attention_rows<DT, DW, NB, NT>, lds);
    if (e != hipSuccess) return e;
    const uint64_t grid = (uint64_t) attention_groups(a, s);
    last_form().grid = grid;
    k_attention_rows<DT, DW, NB, NT><<<dim3((unsigned) grid), dim3(64 * kWaves), lds, stream>>>(a, reinterpret_cast<float *>(scratch), arrive, s.want);
    return hipGetLastError();
}

template <int DT, int NT>
hipError_t by_dim(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    if (a.D <= 64)
        return s.nb == 1 ? go<DT, 64, 1, NT>(a, s, scratch, arrive, stream) : s.nb == 2 ? go<DT, 64, 2, NT>(a, s, scratch, arrive, stream) : go<DT, 64, 4, NT>(a, s, scratch, arrive, stream);
    if (a.D <= 96)
        return s.nb == 1 ? go<DT, 96, 1, NT>(a, s, scratch, arrive, stream) : s.nb == 2 ? go<DT, 96, 2, NT>(a, s, scratch, arrive, stream) : go<DT, 96, 4, NT>(a, s, scratch, arrive, stream);
    if (a.D <= 128)
        return s.nb == 1 ? go<DT, 128, 1, NT>(a, s, scratch, arrive, stream) : s.nb == 2 ? go<DT, 128, 2, NT>(a, s, scratch, arrive, stream) : go<DT, 128, 4, NT>(a, s, scratch, arrive, stream);
    return go<DT, 256, 1, NT>(a, s, scratch, arrive, stream);
}

// 16-bit results take weights of two terms: few rows wait for memory, and with one the result's error would
// be 20 to 40% above that of its own rounding (one token over 900, 64 over up to 8000, two over 131071: the same
// with one term; 64 rows of one request over 60000 keys 105 us with one, 109 with two)
template <int DT>
hipError_t by_result(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    return a.out_type == F32 ? by_dim<DT, kTerms<DT>>(a, s, scratch, arrive, stream) : by_dim<DT, 2>(a, s, scratch, arrive, stream);
}

} // namespace

hipError_t launch_attention_rows(const AttnLaunch & a, const AttnShape & s, uint8_t * scratch, uint32_t * arrive, hipStream_t stream) {
    return a.dtype == F16 ? by_result<F16>(a, s, scratch, arrive, stream) : by_result<BF16>(a, s, scratch, arrive, stream);
}

} // namespace sgk
