// qtopk.hip -- the key blocks each query token reads, by the dot product with pooled keys (gfx950).
//
// Row (b, n, h) = query token n and kv head h:
//   score[u] = sum over the G query heads g of h's group of  q[b, n, h G + g] . k_cmp[b, u, h]
// and the row's blocks are the K largest scores, ties to the lower block, written in ascending
// block order, -1 past the last; blocks that the mask leaves out are never taken.
//
// The selection is that of the exact scores (bf16 products are exact in fp64, whose sums here
// round at 2^-53), although they are computed on the matrix pipe in fp32: the summed query is
// split in two bf16 (hi + lo, 16 bits), and the result is off by at most
//   eps = 2^-15 |Q| |k|,  Q[d] = sum_g |q_g[d]|   (2^-18 the split, 128 accumulations at 2^-23, the
//   G - 1 additions; |k| bounded by the largest chunk norms of the blocks).
// With T the K-th largest computed score, a block above T + 2 eps is certainly taken and one below
// T - 2 eps certainly not (the K-th largest is off by at most eps too).  Where more blocks lie
// between than slots are left -- about 1 row in 50 on fields, every row on constant keys -- their
// scores are formed again in fp64, one block per lane, and compared there.  Where |Q| or |k| is not
// within 2^-50 .. 2^60 (infinite keys and rows of zeros among them), squares, products or scores may leave
// fp32 and eps bounds nothing: all of the row's blocks are then compared in fp64 (every row so: 1.9 ms for the
// call below with zeros, 4.7 with an infinite key a head).  A NaN is never taken.
//
// One workgroup = row tiles of 16 query tokens of one kv head.  Its waves form a tile's scores
// S^T = K Q^T of up to 64 PL blocks with v_mfma_f32_16x16x32_bf16 into LDS (16 rows of fp32), then
// each wave takes rows, PL scores per lane in registers.  A value that K of the lanes' largest scores
// reach, found by a few steps of bisection (a compare and a population count each), bounds T from
// below, so the scores from there on hold all K; there are seldom more than a few of them, and up to
// 64 go one to a lane, where each lane counts the larger ones.
//
// Bound by the selection's waits: 49152 tokens with 3 kv heads of 4 query heads and 768 blocks (nside 64),
// 14.5 Gflop of scores and 94 MB, take 123-127 us (134 in a trace, 49 of them for the scores); a wave waits
// for 53 % of its cycles, the vector ALU is active for 37 % and the matrix pipe busy for 7.  K costs a step
// with 64 (one call: 161 us with K 16, 256 with 48, 269 with 56, 965 with 64): a threshold of 64 lane
// maxima leaves more than 64 candidates.  The keys of a chunk stay in registers for as many row tiles as fill the chip
// once and the next tile's queries are loaded during a selection: with one row tile per workgroup,
// keys from L2 for each, the scores alone took 133 us, all of it 196.  Exact bisections in both places
// were 213 us, and bisection over all PL registers, the first form of this kernel, 432.
// More blocks than 64 PL go in chunks: the rows' best K so far join the next chunk's scores.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "bsa_common.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kRows = 16;       // query tokens per workgroup
constexpr int kMaxTopk = 64;

struct QueryTopkParams {
    const bf16_t* q; int64_t q_sb, q_sn, q_sh;
    const bf16_t* k; int64_t k_sb, k_sn, k_sh;
    const uint8_t* mask;        // [B, nb], 0: never taken; or null
    int64_t* out;               // [B, Nq, Hk, K]
    int B, Nq, nb, Hk, G, K;
    int qtiles;
    int per, groups;            // row tiles a workgroup takes, workgroups of a (batch, kv head)
};

// Signed integers in the order of the floats (none is NaN), and back
__device__ __forceinline__ int order_key(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_value(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// max (or min) over the wave, in every lane: DPP steps within 16 lanes, then the swaps of 16- and
// 32-lane halves (of integers: a float's maximum is two instructions and takes no DPP operand)
template <bool MAX>
__device__ __forceinline__ int either(int a, int b) { return MAX ? max(a, b) : min(a, b); }
template <bool MAX, int CTRL>
__device__ __forceinline__ int dpp_either(int x) { return either<MAX>(x, __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true)); }
template <bool MAX>
__device__ __forceinline__ float wave_either(float y) {
    int x = order_key(y);
    x = dpp_either<MAX, 0xb1>(x);    // quad_perm [1,0,3,2]
    x = dpp_either<MAX, 0x4e>(x);    // quad_perm [2,3,0,1]
    x = dpp_either<MAX, 0x141>(x);   // row_half_mirror
    x = dpp_either<MAX, 0x140>(x);   // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = either<MAX>((int)a[0], (int)a[1]);
    const auto c = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return key_value(__builtin_amdgcn_readfirstlane(either<MAX>((int)c[0], (int)c[1])));
}
__device__ __forceinline__ float wave_max(float x) { return wave_either<true>(x); }
__device__ __forceinline__ float wave_min(float x) { return wave_either<false>(x); }

__device__ __forceinline__ int lanes_from(float x, float t) { return (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(x >= t)); }

// A value that at least K, and where it can be found so soon no more than `most`, of the lanes' values
// (-inf among them; none is NaN) reach, by bisection: a compare and a population count per step.
// -inf where fewer than K are above it.
__device__ __forceinline__ float reached_by(float x, int K, int most) {
    if (lanes_from(x, -__FLT_MAX__) < K) return -INFINITY;
    float hi = wave_max(x), lo = wave_min(x == -INFINITY ? INFINITY : x);
    if (lanes_from(x, hi) >= K) return hi;
    for (;;) {   // lo is reached by K or more, hi by fewer
        const float mid = 0.5f * lo + 0.5f * hi;
        if (!(mid > lo && mid < hi)) return lo;   // neighbours
        const int n = lanes_from(x, mid);
        if (n >= K) {
            lo = mid;
            if (n <= most) return lo;
        } else {
            hi = mid;
        }
    }
}

// The larger of three; a NaN among them does not count (v_max3_f32 alone: the compiler would put a
// canonicalising instruction before each operand)
__device__ __forceinline__ float larger(float a, float b, float c) {
    float y;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
    return y;
}

// A norm, from its square, that eps bounds errors by, or infinity for any other (see above; a NaN is another).
// (The instruction's root is off by one step at most, which eps has room for: the terms above are 1.4 2^-16.)
__device__ __forceinline__ float norm_bound(float square) {
    const float x = __builtin_amdgcn_sqrtf(square);
    return x >= 0x1p-50f && x <= 0x1p60f ? x : INFINITY;
}

// Lane of the n-th set bit of m (anything past the last)
__device__ __forceinline__ int nth_bit(uint64_t m, int n) {
    for (int i = 0; i < n; ++i) m &= m - 1;
    return m == 0 ? 0 : (int)__builtin_ctzll(m);
}

// The exact summed query of a row, a dim per lane, to LDS
__device__ __forceinline__ void summed_query(const QueryTopkParams& p, int b, int n, int h, int lane, double* qs) {
    const bf16_t* qb = p.q + b * p.q_sb + (int64_t)n * p.q_sn + (int64_t)h * p.G * p.q_sh + lane;
    double sum = 0.0;
    for (int g = 0; g < p.G; ++g) sum += (double)bf2f(qb[g * p.q_sh]);
    qs[lane] = sum;
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ double exact_score(const bf16_t* kr, const double* qs) {
    double s[4] = {};   // (one chain of 64 sums would be waited for)
#pragma unroll
    for (int d = 0; d < 64; d += 8) {
        const uint4 w4 = ld16(kr + d);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = fma(qs[d + 2 * j], (double)bf_lo(w[j]), s[j]);
            s[j] = fma(qs[d + 2 * j + 1], (double)bf_hi(w[j]), s[j]);
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}
// x of lane j, the same j in all lanes
__device__ __forceinline__ double lane_value(double x, int j) {
    const uint2 w = __builtin_bit_cast(uint2, x);
    const uint2 y = make_uint2(__builtin_amdgcn_readlane(w.x, j), __builtin_amdgcn_readlane(w.y, j));
    return __builtin_bit_cast(double, y);
}

// How many of the lanes in `of` come before this one: a larger score, or the same and a lower lane.
__device__ __forceinline__ int exact_rank(double x, bool of, int lane) {
    int rank = 0;
    for (uint64_t m = __builtin_amdgcn_ballot_w64(of); m != 0; m &= m - 1) {
        const int j = (int)__builtin_ctzll(m);
        const double y = lane_value(x, j);
        rank += y > x || (y == x && j < lane);
    }
    return rank;
}

// How many values of the lanes in `of` are above y, or equal where `ties`.
__device__ __forceinline__ int exact_above(double x, bool of, double y, bool ties) {
    int n = 0;
    for (uint64_t m = __builtin_amdgcn_ballot_w64(of); m != 0; m &= m - 1) {
        const double z = lane_value(x, (int)__builtin_ctzll(m));
        n += z > y || (ties && z == y);
    }
    return n;
}

// PL = 12 at most: two workgroups of 8 waves fill a CU at 4 waves per SIMD, whose 128 registers hold no
// longer chunk (the whole one of 8 waves spills four, 20 bytes of scratch a lane; LDS would allow 16).
// WHOLE: nb <= 64 PL, one chunk, whose keys stay in registers for all of a workgroup's tiles.
template <int PL, int NW, bool WHOLE>
__global__ __launch_bounds__(NW * 64, 4) void query_topk_kernel(QueryTopkParams p) {
    constexpr int kChunk = 64 * PL, kStride = kChunk + 4;
    static_assert(4 * 64 + 2 * 64 * (PL + 1) <= 4 * kStride, "64 scores and a row's codes fit its scores' place");
    __shared__ __attribute__((aligned(16))) float sc[kRows * kStride];
    constexpr int kCarry = WHOLE ? 1 : kRows;
    __shared__ float carry_v[kCarry][kMaxTopk];   // best K of the chunks so far, ascending blocks
    __shared__ int carry_u[kCarry][kMaxTopk];
    __shared__ int carry_n[kCarry];
    __shared__ float qnorms[2][kRows], knorm[NW];
    __shared__ __attribute__((aligned(16))) bf16_t qpart[2][kRows][72];   // (rows 144 bytes apart: distinct banks)
    __shared__ double qd[NW][64];                // a wave's exact summed query (rows that need it)

    const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = blockIdx.x % p.groups, rest = blockIdx.x / p.groups;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const bf16_t* kb = p.k + b * p.k_sb + h * p.k_sh;
    const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (int64_t)b * p.nb;

    // a wave's tiles of 16 blocks of a chunk, every NW-th
    constexpr int kTiles = 4 * PL / NW;
    static_assert(kTiles * NW == 4 * PL, "the waves share a chunk's tiles evenly");
    uint4 a[kTiles][2];
    uint32_t ons[kTiles];   // the flag of block c of a tile is bit c
    float kn = -1.f;        // largest squared norm of this lane's dims over the blocks it has loaded (-1: none)
    auto load_keys = [&](int u0) {
        bool on[kTiles];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            const int u = u0 + 16 * (wave + j * NW) + c16, at = min(u, p.nb - 1);
            const bf16_t* kr = kb + (int64_t)at * p.k_sn + 8 * g4;
            a[j][0] = ld16(kr);
            a[j][1] = ld16(kr + 32);
            on[j] = u < p.nb;
            if (mask != nullptr) on[j] = on[j] && mask[at];
        }
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
            float nn = 0.f;
            const uint32_t aw[8] = {a[j][0].x, a[j][0].y, a[j][0].z, a[j][0].w, a[j][1].x, a[j][1].y, a[j][1].z, a[j][1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bf16x2 e = __builtin_bit_cast(bf16x2, aw[i]);
                nn = __builtin_amdgcn_fdot2_f32_bf16(e, e, nn, false);
            }
            kn = on[j] ? fmaxf(kn, nn) : kn;
            ons[j] = (uint32_t)__builtin_amdgcn_ballot_w64(on[j]);
        }
        // |k|^2 <= the sum over the four dim groups of their largest
        float m = kn;
        int key = __float_as_int(m);   // (of one negative value: in order as they are)
        key = dpp_either<true, 0xb1>(key);
        key = dpp_either<true, 0x4e>(key);
        key = dpp_either<true, 0x141>(key);
        m = __int_as_float(dpp_either<true, 0x140>(key));
        m += __shfl_xor(m, 16);
        m += __shfl_xor(m, 32);
        if (lane == 0) knorm[wave] = m;
    };

    // the summed queries of a row tile, each thread a run of dims of one; the first heads' dims are
    // loaded a tile ahead
    constexpr int kDims = kRows * 64 / (NW * 64), kLanes = 64 / kDims;   // dims a thread, threads a query
    static_assert(kDims == 2 || kDims == 1, "one or two dims a thread");
    const int qr = threadIdx.x / kLanes, qdim = threadIdx.x % kLanes * kDims;
    auto query = [&](int tile) {
        return p.q + b * p.q_sb + (int64_t)min(tile * kRows + qr, p.Nq - 1) * p.q_sn + (int64_t)h * p.G * p.q_sh + qdim;
    };
    auto dims = [&](const bf16_t* x) { return kDims == 2 ? *reinterpret_cast<const uint32_t*>(x) : (uint32_t)*x; };
    constexpr int kAhead = 4;
    uint32_t ahead[kAhead];
    auto load_queries = [&](int tile) {
        const bf16_t* qb = query(tile);
#pragma unroll
        for (int g = 0; g < kAhead; ++g) ahead[g] = dims(qb + min(g, p.G - 1) * p.q_sh);
    };

    const int first = grp * p.per, past = min(first + p.per, p.qtiles);
    load_queries(first);
    if constexpr (WHOLE) load_keys(0);
    for (int tile = first; tile < past; ++tile) {
        const int n0 = tile * kRows, rows = min(kRows, p.Nq - n0);
        float* qnorm = qnorms[tile & 1];   // (waves still selecting read the last tile's)
        {   // as hi + lo parts by way of LDS
            float sum[kDims] = {}, tot[kDims] = {};
            auto add = [&](uint32_t w) {
                const float x[2] = {bf_lo(w), bf_hi(w)};
#pragma unroll
                for (int i = 0; i < kDims; ++i) {
                    sum[i] += x[i];
                    tot[i] += fabsf(x[i]);
                }
            };
#pragma unroll
            for (int g = 0; g < kAhead; ++g)
                if (g < p.G) add(ahead[g]);
            if (p.G > kAhead) {
                const bf16_t* qb = query(tile);
#pragma unroll 4
                for (int g = kAhead; g < p.G; ++g) add(dims(qb + g * p.q_sh));
            }
            float mag = 0.f;
#pragma unroll
            for (int i = 0; i < kDims; ++i) {
                const float hi = round_bf16(sum[i]);
                qpart[0][qr][qdim + i] = (bf16_t)(__float_as_uint(hi) >> 16);
                qpart[1][qr][qdim + i] = (bf16_t)(pack_bf16x2(sum[i] - hi, 0.f) & 0xffffu);
                mag = fmaf(tot[i], tot[i], mag);
            }
#pragma unroll
            for (int m = 1; m < kLanes; m <<= 1) mag += __shfl_xor(mag, m);
            if (threadIdx.x % kLanes == 0) qnorm[qr] = norm_bound(mag);
        }
        __syncthreads();
        bf16x8 hi[2], lo[2];   // of column c16, dims 32 ks + 8 g4 .. + 7
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            hi[ks] = as_bf16x8(*reinterpret_cast<const uint4*>(&qpart[0][c16][32 * ks + 8 * g4]));
            lo[ks] = as_bf16x8(*reinterpret_cast<const uint4*>(&qpart[1][c16][32 * ks + 8 * g4]));
        }
        for (int u0 = 0; u0 < (WHOLE ? 1 : p.nb); u0 += kChunk) {
            if constexpr (!WHOLE) load_keys(u0);
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
                s = mfma16(as_bf16x8(a[j][0]), hi[0], s);
                s = mfma16(as_bf16x8(a[j][1]), hi[1], s);
                if (p.G > 1) {
                    s = mfma16(as_bf16x8(a[j][0]), lo[0], s);
                    s = mfma16(as_bf16x8(a[j][1]), lo[1], s);
                }
                // lane: blocks 16 t + 4 g4 + e of query c16; -inf where there is none or the mask leaves it out
                float4 v = make_float4(s[0], s[1], s[2], s[3]);
                uint32_t bits = ons[j];
                asm volatile("" : "+s"(bits));   // (the tests of all tiles would be held in registers otherwise)
                if (bits != ~0u) {
                    const uint32_t four = bits >> (4 * g4);
                    v.x = (four & 1) ? v.x : -INFINITY;
                    v.y = (four & 2) ? v.y : -INFINITY;
                    v.z = (four & 4) ? v.z : -INFINITY;
                    v.w = (four & 8) ? v.w : -INFINITY;
                }
                *reinterpret_cast<float4*>(sc + c16 * kStride + 16 * (wave + j * NW) + 4 * g4) = v;
            }
            __syncthreads();
            const bool last = WHOLE || u0 + kChunk >= p.nb;
            if (last && tile + 1 < past) load_queries(tile + 1);
            float kmax = knorm[0];
#pragma unroll
            for (int i = 1; i < NW; ++i) kmax = fmaxf(kmax, knorm[i]);
            kmax = kmax < 0.f ? 1.f : norm_bound(kmax);   // (no block yet, and so no score)
            // row r's blocks, ascending by lane
            auto store = [&](int r, bool take, int u, float mine) {
                const uint64_t m = __builtin_amdgcn_ballot_w64(take);
                const int count = (int)__builtin_popcountll(m);
                const int pos = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
                asm volatile("" ::: "memory");         // the carried blocks are read before they are written
                if (WHOLE || last) {
                    int64_t* row = p.out + (((int64_t)b * p.Nq + n0 + r) * p.Hk + h) * p.K;
                    if (take && pos < p.K) row[pos] = u;
                    if (lane >= count && lane < p.K) row[lane] = -1;
                } else {
                    if (take) {
                        carry_v[r][pos] = mine;
                        carry_u[r][pos] = u;
                    }
                    if (lane == 0) carry_n[r] = count;
                }
            };
            // A row's best K by exact scores, one a lane and ascending: hold(there, u) adds the lanes' blocks that
            // are there, all of them above the held ones.  A NaN is not held.
            double held, lowest;   // (lowest: of K held ones, which a further one has to exceed)
            int held_u, holds;
            auto hold_none = [&](int r) {
                summed_query(p, b, n0 + r, h, lane, qd[wave]);
                held = lowest = -INFINITY;
                held_u = holds = 0;
            };
            auto hold = [&](bool there, int fu) {
                const double x = there ? exact_score(kb + (int64_t)fu * p.k_sn, qd[wave]) : -INFINITY;
                const bool fresh = there && x == x && (holds < p.K || x > lowest), old = lane < holds;
                if (__builtin_amdgcn_ballot_w64(fresh) == 0) return;
                const int rank_x = exact_rank(x, fresh, lane) + exact_above(held, old, x, true);
                const int rank_h = exact_rank(held, old, lane) + exact_above(x, fresh, held, false);
                const uint64_t mh = __builtin_amdgcn_ballot_w64(old && rank_h < p.K);
                const uint64_t mx = __builtin_amdgcn_ballot_w64(fresh && rank_x < p.K);
                const int nh = (int)__builtin_popcountll(mh);
                const int jh = nth_bit(mh, min(lane, 63)), jx = nth_bit(mx, max(lane - nh, 0));
                const double before = held, h1 = __shfl(held, jh), x1 = __shfl(x, jx);
                const int u1 = __shfl(held_u, jh), u2 = __shfl(fu, jx);
                held = lane < nh ? h1 : x1;
                held_u = lane < nh ? u1 : u2;
                holds = nh + (int)__builtin_popcountll(mx);
                if (holds == p.K) {
                    const uint64_t lx = __builtin_amdgcn_ballot_w64(fresh && rank_x == p.K - 1), lh = __builtin_amdgcn_ballot_w64(old && rank_h == p.K - 1);
                    lowest = lx != 0 ? lane_value(x, (int)__builtin_ctzll(lx)) : lane_value(before, (int)__builtin_ctzll(lh));
                }
            };
            uint32_t open_rows = 0;   // those without a bound
            for (int r = wave; r < rows; r += NW) {
                const float e2 = 0x1p-14f * qnorm[r] * kmax;   // 2 eps
                if (__builtin_amdgcn_ballot_w64(e2 < INFINITY) == 0) {
                    open_rows |= 1u << r;
                    continue;
                }
                // element 0: the carried best, element 1 + i: block u0 + lane + 64 i; -inf where there is none
                float v[PL + 1];
                v[0] = !WHOLE && u0 > 0 && lane < carry_n[r] ? carry_v[r][lane] : -INFINITY;
#pragma unroll
                for (int i = 0; i < PL; ++i) v[1 + i] = sc[r * kStride + lane + 64 * i];
                static_assert(PL % 2 == 0, "pairs of scores");
                float top = larger(v[0], v[1], v[2]);
#pragma unroll
                for (int i = 3; i < PL; i += 2) top = larger(top, v[i], v[i + 1]);
                top = larger(top, v[PL], -INFINITY);         // (where all of them are NaN)
                // Where K of the lanes' largest scores reach a value, T is no smaller.  Scores within 2 eps of
                // it go one to a lane, ascending by block, where they are no more than 64: nearly always where
                // K is no more than half the lanes; else the value is raised first.
                float least = reached_by(top, p.K, max(p.K, min(p.K + 8, 32)));
                auto all_from = [&](float t) {
                    int n = 0;
#pragma unroll
                    for (int i = WHOLE; i <= PL; ++i) n += lanes_from(v[i], t);
                    return n;
                };
                if (p.K > 24 && all_from(fmaxf(least - e2, -__FLT_MAX__)) > 64) {
                    float lo = least == -INFINITY ? wave_min(top == -INFINITY ? INFINITY : top) : least, hi = wave_max(top);
                    for (;;) {
                        const float mid = 0.5f * lo + 0.5f * hi;
                        if (!(mid > lo && mid < hi)) break;
                        const int n = all_from(mid);
                        if (n < p.K) {
                            hi = mid;
                            continue;
                        }
                        lo = least = mid;
                        if (n <= 64 && all_from(mid - e2) <= 64) break;
                    }
                }
                const float keep = fmaxf(least - e2, -__FLT_MAX__);
                float* scores = sc + r * kStride;                            // of the first 64, and all codes
                uint16_t* codes = reinterpret_cast<uint16_t*>(scores + 64);   // (64 i + l: element i of lane l)
                asm volatile("" ::: "memory");     // the row's scores are read before these take their place
                scores[lane] = -INFINITY;
                int n = 0;
#pragma unroll
                for (int i = WHOLE; i <= PL; ++i) {
                    const uint64_t m = __builtin_amdgcn_ballot_w64(v[i] >= keep);
                    if (m == 0) continue;
                    const int pos = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, (uint32_t)n));
                    n += (int)__builtin_popcountll(m);
                    if (v[i] >= keep) {
                        codes[pos] = (uint16_t)(64 * i + lane);
                        if (n <= 64) scores[pos] = v[i];   // (of more than 64 nobody reads them)
                    }
                }
                asm volatile("" ::: "memory");     // (LDS is in order within a wave)
                auto block = [&](int code) { return !WHOLE && code < 64 ? carry_u[r][code] : u0 + code - 64; };
                bool take;
                float mine = -INFINITY;
                int u = 0;
                if (n <= 64) {
                    take = lane < n;
                    if (take) {
                        u = block(codes[lane]);
                        mine = scores[lane];
                    }
                    if (n > p.K) {
                        // T is the smallest that has fewer than K above it
                        int above = 0;
                        for (int i = 0; i < n; i += 8) {
                            const float4 x = *reinterpret_cast<const float4*>(scores + i), y = *reinterpret_cast<const float4*>(scores + i + 4);
                            above += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
                            above += (y.x > mine) + (y.y > mine) + (y.z > mine) + (y.w > mine);
                        }
                        uint64_t at = 0;
                        for (int i = p.K - 1; at == 0; --i) at = __builtin_amdgcn_ballot_w64(take && above == i);   // (equal ones: fewer)
                        const float T = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), (int)__builtin_ctzll(at)));
                        const uint64_t in = __builtin_amdgcn_ballot_w64(mine >= T - e2 && lane < n);
                        take = in >> lane & 1;
                        if ((int)__builtin_popcountll(in) > p.K) {
                            // more within 2 eps of T than slots are left: exact scores decide
                            const bool open = take && mine <= T + e2;
                            take = take && !open;
                            const int sure = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(take));
                            summed_query(p, b, n0 + r, h, lane, qd[wave]);
                            const double x = open ? exact_score(kb + (int64_t)u * p.k_sn, qd[wave]) : -INFINITY;
                            const int rank = exact_rank(x, open, lane);
                            take = take || (open && rank < p.K - sure);
                        }
                    }
                } else {
                    // ties: all candidates, 64 at a time
                    hold_none(r);
                    for (int at = 0; at < n; at += 64) hold(at + lane < n, at + lane < n ? block(codes[at + lane]) : 0);
                    take = lane < holds;
                    u = held_u;
                    mine = (float)held;
                }
                store(r, take, u, mine);
            }
            for (; open_rows != 0; open_rows &= open_rows - 1) {   // all blocks
                const int r = (int)__builtin_ctz(open_rows);
                hold_none(r);
                if (!WHOLE && u0 > 0) hold(lane < carry_n[r], lane < carry_n[r] ? carry_u[r][lane] : 0);
                for (int u = u0; u < min(u0 + kChunk, p.nb); u += 64)
                    hold(u + lane < p.nb && (mask == nullptr || mask[u + lane]), min(u + lane, p.nb - 1));
                store(r, lane < holds, held_u, (float)held);
            }
            if (!last) __syncthreads();   // the rows' scores are read before the next chunk's are written
        }
    }
}

template <int PL, bool WHOLE>
const void* topk_fn(bool wide) {
    return wide ? (const void*)&query_topk_kernel<PL, 16, WHOLE> : (const void*)&query_topk_kernel<PL, 8, WHOLE>;
}

bool rows_ok(const mosaic_bnhd& t) {
    return (reinterpret_cast<uintptr_t>(t.ptr) & 15u) == 0 && t.stride_b % 8 == 0 && t.stride_n % 8 == 0 && t.stride_h % 8 == 0;
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" int mosaic_query_topk_fwd(mosaic_bnhd q, mosaic_bnhd k_cmp, const uint8_t* block_mask, int32_t batch,
                                     int32_t num_queries, int32_t num_blocks, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t block_count,
                                     int64_t* indices_out, void* stream) {
    if (batch <= 0 || num_queries <= 0 || num_blocks <= 0) return MOSAIC_ERR_SHAPE;
    if (head_dim != kHeadDim) return MOSAIC_ERR_HEAD_DIM;
    if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return MOSAIC_ERR_HEADS;
    if (num_q_heads / num_kv_heads > 16) return MOSAIC_ERR_UNSUPPORTED;
    if (block_count <= 0 || block_count > num_blocks) return MOSAIC_ERR_BLOCK_COUNT;
    if (block_count > kMaxTopk) return MOSAIC_ERR_UNSUPPORTED;
    if (q.ptr == nullptr || k_cmp.ptr == nullptr || indices_out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!rows_ok(q) || !rows_ok(k_cmp) || (reinterpret_cast<uintptr_t>(indices_out) & 7u)) return MOSAIC_ERR_ALIGNMENT;
    QueryTopkParams p{};
    p.q = static_cast<const bf16_t*>(q.ptr); p.q_sb = q.stride_b; p.q_sn = q.stride_n; p.q_sh = q.stride_h;
    p.k = static_cast<const bf16_t*>(k_cmp.ptr); p.k_sb = k_cmp.stride_b; p.k_sn = k_cmp.stride_n; p.k_sh = k_cmp.stride_h;
    p.mask = block_mask;
    p.out = indices_out;
    p.B = batch; p.Nq = num_queries; p.nb = num_blocks; p.Hk = num_kv_heads; p.G = num_q_heads / num_kv_heads; p.K = block_count;
    p.qtiles = (int)(((int64_t)num_queries + kRows - 1) / kRows);
    const int64_t wgs = (int64_t)p.qtiles * num_kv_heads * batch;
    if (wgs > 0x7fffffff) return MOSAIC_ERR_SHAPE;
    const bool wide = wgs < 256;
    const void* fn = num_blocks <= 256   ? topk_fn<4, true>(wide)
                     : num_blocks <= 512 ? topk_fn<8, true>(wide)
                     : num_blocks <= 768 ? topk_fn<12, true>(wide)
                                         : topk_fn<12, false>(wide);
    // Two workgroups are resident on a CU.  Each takes as many row tiles of its kv head as fill the chip
    // once, so that keys (of one chunk) are loaded once; about four times where kv heads are many.
    const int64_t heads = (int64_t)num_kv_heads * batch, want = (heads <= 64 ? 512 : 2048) / heads;
    p.per = (int)(want < 1 ? p.qtiles : ((int64_t)p.qtiles + want - 1) / want);
    p.groups = (p.qtiles + p.per - 1) / p.per;
    void* args[] = {&p};
    return hipLaunchKernel(fn, dim3((unsigned)(p.groups * heads)), dim3(wide ? 1024 : 512), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess
               ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}
