// cattn.hip -- attention of query tokens over a key/value cache held in 8 bits (gfx950).
//
// Row (b, n, g) = query token n and query head g of kv head h; over its keys u, those below the
// sequence's length and, where the call names key blocks, of the token's blocks:
//   o = sum_u p_u v_u / sum_u p_u,  p_u = exp2(c q.k_u - m),  c = softmax_scale log2 e,
//   k_u = ks code, v_u = vs code, ks and vs the scales of u's block and head
// Codes are whole numbers of at most 8 bits or e4m3, exact in bf16, so the products are of bf16 operands
// without a rounding of theirs.  ks goes into the factor of the scores and vs into the exponent,
//   P = exp2(c ks q.code_k - m + log2(vs / w)),  O = sum P code_v,  l = sum P w / vs,  o = w O / l,
// so that neither costs an instruction per score (w: the scale of the sequence's first block).  fp32 scores,
// maxima, sums and accumulators.  P is rounded to bf16 for the product with the values and l sums the rounded P:
// an error as the output's own rounding (together 2.2e-3 of the result, the output's alone 1.7e-3); a second term of
// P would be half as many products again where they are the bound.  Of few rows it is taken: see there.
//
// Two kernels.  Many rows: a workgroup takes 4 or 12 waves x QW = 32 / G tokens of one kv head, a wave the 32 rows
// (token, head) of its tokens; the codes of 64 keys are converted once, by all of its waves, into operand order in
// LDS, which each of them reads.  12 heads of 12288 tokens over 49152 keys, 1.86 TFLOP: 1.65 to 1.77 ms, 1050 to 1130
// TF/s, where a bf16 library product of 8192^3 reaches 1200 to 1230 under the same power limit (1.9 GHz: vector ALU 66 %
// of the cycles, matrix pipe 48 %).  With blocks for each token (49152 tokens, 16 blocks of 64, 12 heads: 0.21 to 0.23
// ms, 660 to 730 TF/s; 65 % and 32 %) a workgroup walks the union of its tokens' blocks: a quarter of its 67000 cycles
// goes before the first tile, into the union and its scales.
// Few rows (up to 16 of a kv head, one token above all): memory bounds a long cache (one token over 196608 keys of 3
// heads in e4m3, 75 MB: 15.5 us, 4.9 TB/s), the vector ALU's conversions and the launch a short one.
// In both, the keys of a call with few workgroups are split into shares, and a third kernel joins their parts.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "bsa_common.h"
#include "lds_dma.h"
#include "mosaic_bsa.h"
#include "qcache.h"
#include "query_rows.h"

namespace mosaic {
namespace {

struct CacheAttnParams : QuerySets {
    mosaic_kv_cache cache;
    const bf16_t* q; int64_t q_sb, q_sn, q_sh;
    bf16_t* out;               // [B, Nq, Hq, 64]
    float* part_o;             // [splits, parts, 64] (splits > 1): o of a split's keys
    float2* part_ml;           // [splits, parts] (m, l): 2^m l is the sum of its weights
    int64_t* part_at;          // [parts] the row that a part belongs to, or -1
    int64_t parts;             // rows that are joined
    int whole;                 // tiles of rows that one workgroup takes with all of their keys
    float c;
};

// A tile of 64 keys in operand order: keys [kt 2][step 4][lane 64][8], values [kt 2][dt 2][step 2][lane 64][8]
struct CacheTile {
    __attribute__((aligned(1024))) bf16_t K[64 * 64];
    __attribute__((aligned(1024))) bf16_t V[64 * 64];
};
struct DenseLds { CacheTile tile[2]; };
struct SetsLds : UnionLds { CacheTile tile[2]; };

struct AttnState {
    f32x16 o[2];      // O^T [dim tile]
    float m, l;       // reference of the scores, and this lane's part of the sum
    float c;          // SAFE: the factor of the row's scores
    bool has;         // a key above -inf was met
    bool wide;        // so was a scale of values, or a query, that SAFE is for
};

// How a tile is computed.  attend_whole: no score exceeds kBound (|q| and the blocks' norms say so), and the
// reference is 0.  attend_tile: it is 0 too unless a score leaves +- kBound, and moves then, so that a row's bits
// do not depend on the form, and on the rows beside it only where a union without an order is cut into shares, by its size.
// Which form is one decision for a wave's rows and up to 64 blocks (12288 tokens over 49152 keys: 1720 us, 1780 where one
// token of 100 leaves the bound, 1910 to 1960 where all or a block of each 64 do; the tokens of nside 64 with blocks of
// their own 213, 211 and 222 to 227).  SAFE: for rows that end with a value that is not
// finite or with a reference past kFar, for scales of values further than kSpread from w, and for queries of a norm of 2^63 or
// more: the reference is the maximum, and a row's accumulators take nothing from a block that it has not, not even 0 * NaN.
// A query with an element of 2^80 or more goes into it times 2^-32, and its scores' factor times 2^32: with codes in the
// place of keys its products would leave fp32 where the scores do not.
// With these P is 2^-100 at least, 26 bits above the smallest normal number; an overflow of its sums ends in SAFE.
// An underflow does not show, so it is kept away: a fused score differs from its maximum, a rounded product, by half a
// unit of the reference, and lv - m is rounded to one; up to kFar that is 2^-9, what P's own rounding is, but of scores past
// 2^30 it leaves the largest P anywhere from 0 to infinity.
constexpr float kBound = 80.f;
constexpr float kSpread = 0x1p20f;
constexpr float kFar = 0x1p15f;
constexpr float kLargeQuery = 0x1p126f;                  // (the norm's square)
constexpr uint16_t kLargeElement = (127 + 80) << 7;      // (bf16's bits)

// x a + b in two roundings
__device__ __forceinline__ float times_plus(float x, float a, float b) {
#pragma clang fp contract(off)
    const float y = x * a;
    return y + b;
}

// Scores of tokens at or past `left` of a lane's 16 become -inf
__device__ __forceinline__ void mask_scores(f32x16& s, int left) {
    asm volatile("" : "+v"(left));   // (opaque, or the comparisons of all calls are kept at once)
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = e < left ? s[e] : -INFINITY;
}

// P of 8 scores, as an operand
template <bool SAFE>
__device__ __forceinline__ bf16x8 weights(const f32x16& s, int s2, float ck, float ref) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = s[8 * s2 + 2 * i], y = s[8 * s2 + 2 * i + 1];
        // (in SAFE the score at the maximum is the maximum, whatever its unit: P is 1 there)
        w[i] = SAFE ? pack_bf16x2(__builtin_amdgcn_exp2f(times_plus(x, ck, ref)), __builtin_amdgcn_exp2f(times_plus(y, ck, ref)))
                          : pack_bf16x2(__builtin_amdgcn_exp2f(fmaf(x, ck, ref)), __builtin_amdgcn_exp2f(fmaf(y, ck, ref)));
    }
    return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
}

// What the scales of values are taken relative to: that of the sequence's first block (1 where that is zeros or
// not finite), so that it does not depend on what else a workgroup computes.  Rows without that block follow it by their
// roundings in fp32, and beyond kSpread by the second pass.
__device__ __forceinline__ float value_unit(const mosaic_kv_cache& c, int b, int h) {
    const float vs = c.v_scale[block_at(c, b, 0, h)];
    return vs > 0.f && vs < INFINITY ? vs : 1.f;
}

// c ks as an fp32 number above 0
__device__ __forceinline__ float score_factor(float c, float ks) { return fminf(fmaxf(c * ks, FLT_MIN), FLT_MAX); }

// Factors of a block's scales: scores by ck = c ks; P times 2^lv = vs / w, and iv = w / vs for the sum of P (SAFE:
// ck = ks, as c is a row's own, lv = vs itself, iv an addend of the scores that is 0 or NaN).  A scale of 0 stands for
// zeros only: any positive one does.  A NaN among them goes where only the members of the block meet it.
struct Factors { float ck, lv, iv; };
template <bool SAFE>
__device__ __forceinline__ Factors factors(float c, float ks, float vs, float w, bool& wide) {
    Factors f;
    f.ck = ks > 0.f ? (SAFE ? ks : score_factor(c, ks)) : 1.f;
    const float poison = ks - ks;
    wide = false;
    if constexpr (SAFE) {
        f.lv = vs;
        f.iv = poison;
    } else {
        const float ratio = vs * __builtin_amdgcn_rcpf(w);   // (reciprocals to a unit of the last place)
        const bool near = ratio <= kSpread && ratio >= 1.f / kSpread;
        wide = !near && vs != 0.f;   // (a NaN too: SAFE leaves it a NaN)
        const float of = near ? ratio : 1.f;
        f.lv = __builtin_amdgcn_logf(of) + poison;
        f.iv = __builtin_amdgcn_rcpf(of);
    }
    return f;
}

// Whether an element of a query's operand is kLargeElement or more (infinities and NaN too), the factor of the scores of a
// row where one is, and its operands then.  (A factor past fp32, c above 2^96, stays in it: products of 2^48 and more
// are then one key's all the same.)
__device__ __forceinline__ bool large_query(const bf16x8& f) {
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    const u16x8 x = __builtin_bit_cast(u16x8, f) & (uint16_t)0x7fff;
    const auto y = __builtin_elementwise_max(x.lo, x.hi);
    const auto z = __builtin_elementwise_max(y.lo, y.hi);
    return max(z.x, z.y) >= kLargeElement;
}
__device__ __forceinline__ float row_factor(float c, bool large) { return large ? fminf(c * 0x1p32f, FLT_MAX) : c; }
__device__ __forceinline__ bf16x8 within(const bf16x8& f, bool large) {
    const uint4 u = __builtin_bit_cast(uint4, f);
    const float by = large ? 0x1p-32f : 1.f;
    auto times = [&](uint32_t x) { return pack_bf16x2(bf_lo(x) * by, bf_hi(x) * by); };
    return as_bf16x8(make_uint4(times(u.x), times(u.y), times(u.z), times(u.w)));
}

// The first of a share's units, where the first shares take one more
__device__ __forceinline__ int share_begin(int units, int share, int shares) {
    const int each = (int)((uint32_t)units / (uint32_t)shares);
    return each * share + min(share, units - each * shares);
}

struct TileRead {
    const CacheTile& t;
    int lane;
    __device__ __forceinline__ bf16x8 key(int kt, int ds) const { return as_bf16x8(ld16(t.K + ((kt * 4 + ds) * 64 + lane) * 8)); }
    __device__ __forceinline__ bf16x8 val(int kt, int dt, int s2) const { return as_bf16x8(ld16(t.V + (((kt * 2 + dt) * 2 + s2) * 64 + lane) * 8)); }
};

// One tile of 64 keys; valid: how many of them exist.
template <bool SAFE>
__device__ __forceinline__ void attend_tile(const CacheTile& tile, const bf16x8 (&qf)[4], bool member, int valid, const Factors& f, AttnState& a) {
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const TileRead t{tile, lane};
    f32x16 s[2] = {splat(0.f), splat(0.f)};
#pragma unroll
    for (int ds = 0; ds < 4; ++ds)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = mfma32(t.key(kt, ds), qf[ds], s[kt]);
    if (valid < 64) {
        seldom();
        mask_scores(s[0], valid - 16 * hh);
        mask_scores(s[1], valid - 32 - 16 * hh);
    }
    float mt = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mt = __builtin_elementwise_maximum(mt, s[kt][e]);
    const float ck = SAFE ? score_factor(a.c, f.ck) : f.ck;
    mt = xor32_max(mt) * ck;
    const bool some = member && mt > -INFINITY;
    const bool move = some && (SAFE ? !a.has || mt > a.m : mt > a.m + kBound || (!a.has && mt < -kBound));
    if (__builtin_amdgcn_ballot_w64(move)) {
        const float alpha = move && a.has ? __builtin_amdgcn_exp2f(a.m - mt) : 1.f;
        a.m = move ? mt : a.m;
        a.o[0] *= alpha;
        a.o[1] *= alpha;
        a.l *= alpha;
    }
    a.has = a.has || some;
    const float ref = member ? (SAFE ? f.iv : f.lv) - a.m : -INFINITY;   // P = 0 for the others
    bf16x8 pb[2][2];
    float lt = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            pb[kt][s2] = weights<SAFE>(s[kt], s2, ck, ref);
            lt = operand_sum(pb[kt][s2], lt);
        }
    if constexpr (SAFE) {
        if (member) a.l += lt;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            f32x16 y = splat(0.f);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) y = mfma32(t.val(kt, dt, s2), pb[kt][s2], y);
#pragma unroll
            for (int e = 0; e < 16; ++e) a.o[dt][e] = member ? fmaf(y[e], f.lv, a.o[dt][e]) : a.o[dt][e];
        }
    } else {
        a.l = fmaf(lt, f.iv, a.l);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) a.o[dt] = mfma32(t.val(kt, dt, s2), pb[kt][s2], a.o[dt]);
    }
}

// A whole tile of bounded scores, laid out for the matrix pipe and the vector ALU to run side by side within a wave:
// the scores of the first 32 keys, under them the staging of the next tile; those of the others, under them the
// first weights; the product of these, under it the other weights; their product, under what comes next.
template <typename Stage>
__device__ __forceinline__ void attend_whole(const CacheTile& tile, const bf16x8 (&qf)[4], bool member, const Factors& f, AttnState& a, Stage stage) {
    const TileRead t{tile, (int)(threadIdx.x & 63)};
    const float ref = member ? f.lv : -INFINITY;   // P = 0 for the others
    bf16x8 x[4], p[2], w[2];                       // x: operands, the keys', then the values' [s2][dt]
    f32x16 s = splat(0.f), u = splat(0.f);
    float lt = 0.f;
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) x[ds] = t.key(0, ds);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) s = mfma32(x[ds], qf[ds], s);
    __builtin_amdgcn_sched_barrier(0);
    stage();
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) x[ds] = t.key(1, ds);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
        u = mfma32(x[2 * s2], qf[2 * s2], u);
        u = mfma32(x[2 * s2 + 1], qf[2 * s2 + 1], u);
        p[s2] = weights<false>(s, s2, f.ck, ref);
        lt = operand_sum(p[s2], lt);
        x[2 * s2] = t.val(0, 0, s2);
        x[2 * s2 + 1] = t.val(0, 1, s2);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) a.o[dt] = mfma32(x[2 * s2 + dt], p[s2], a.o[dt]);
        w[s2] = weights<false>(u, s2, f.ck, ref);
        lt = operand_sum(w[s2], lt);
        x[2 * s2] = t.val(1, 0, s2);
        x[2 * s2 + 1] = t.val(1, 1, s2);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) a.o[dt] = mfma32(x[2 * s2 + dt], w[s2], a.o[dt]);
    a.l = fmaf(lt, f.iv, a.l);
}

// The loop over the tiles of a workgroup's blocks
template <bool FP8, bool DENSE, bool SAFE, int WAVES, typename Lds>
struct Walk {
    const CacheAttnParams& p;
    Lds& L;
    int b, h, end;
    float w;        // value_unit
    const bf16x8 (&qf)[4];
    const Row& row;
    AttnState& a;

    // The 512 runs of 16 codes of a tile, those of the keys first: a thread stages one of either, of more waves one
    static constexpr int kRuns = WAVES == 4 ? 2 : 1;
    struct Staged { uint4 x[kRuns]; };
    __device__ __forceinline__ static int first_run() { return WAVES == 4 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x) & ~255; }
    __device__ __forceinline__ void load(int block, int st, Staged& r) const {
        if (first_run() >= 512) return;
        const int64_t from = ((int64_t)b * p.nb * p.Hk + h) * (p.bs * 64) + (uint64_t)(uint32_t)block * (uint32_t)(p.Hk * p.bs * 64) + st * kCodeTile;
        const uint32_t at = 16 * (threadIdx.x & 255);
        if constexpr (kRuns == 2) {
            r.x[0] = ld16(static_cast<const uint8_t*>(p.cache.k_codes) + from + at);
            r.x[1] = ld16(static_cast<const uint8_t*>(p.cache.v_codes) + from + at);
        } else r.x[0] = ld16(static_cast<const uint8_t*>(first_run() == 0 ? p.cache.k_codes : p.cache.v_codes) + from + at);
    }
    __device__ __forceinline__ static void expand(bf16_t* at, const uint4& u) {   // 16 codes: two operands of a lane
        const uint2 a = codes_bf16<FP8>(u.x), b = codes_bf16<FP8>(u.y), c = codes_bf16<FP8>(u.z), d = codes_bf16<FP8>(u.w);
        *reinterpret_cast<uint4*>(at) = make_uint4(a.x, a.y, b.x, b.y);
        *reinterpret_cast<uint4*>(at + 64 * 8) = make_uint4(c.x, c.y, d.x, d.y);
    }
    __device__ __forceinline__ void put(int buf, const Staged& r) const {
        const int tid = threadIdx.x, at = ((tid >> 6 & 3) * 2 * 64 + (tid & 63)) * 8;
        if (first_run() >= 512) return;
        if constexpr (kRuns == 2) {
            expand(L.tile[buf].K + at, r.x[0]);
            expand(L.tile[buf].V + at, r.x[1]);
        } else expand((first_run() == 0 ? L.tile[buf].K : L.tile[buf].V) + at, r.x[0]);
    }
    // |q|^2 of the lane's row
    __device__ __forceinline__ float norm_square() const {
        float square = 0.f;
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) {
            const uint4 u = __builtin_bit_cast(uint4, qf[ds]);
            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) square = fmaf(bf_lo(x[i]), bf_lo(x[i]), fmaf(bf_hi(x[i]), bf_hi(x[i]), square));
        }
        return xor32_add(square);
    }
    // c |q| of the wave's rows at most, a little more than its roundings (a NaN stays).  Elements below 2^-63, whose squares
    // leave fp32, add 8 * 2^-63 to |q| at most: nothing beside 80 but where c is large.
    __device__ __forceinline__ float bound(float square) const { return (sqrtf(wave_max_nonneg(square)) + 0x1p-60f) * p.c * 1.001f; }
    // up to 64 blocks, lane i < count holding the i-th and its members among the wave's tokens
    __device__ __forceinline__ void blocks(int count, int block, int members) {
        const int64_t at = block_at(p.cache, b, block, h);
        const float ks = p.cache.k_scale[at], vs = p.cache.v_scale[at], norm = p.cache.k_norm[at];
        Staged r;
        load(__builtin_amdgcn_readlane(block, 0), 0, r);
        bool wide;
        const Factors f = factors<SAFE>(p.c, ks, vs, w, wide);
        bool bounded = false;
        if constexpr (!SAFE) {
            for (uint64_t far = __builtin_amdgcn_ballot_w64(wide); far != 0; far &= far - 1)
                a.wide = a.wide || DENSE || row.in((uint32_t)__builtin_amdgcn_readlane(members, (int)__builtin_ctzll(far)));
            const float square = norm_square();
            a.wide = a.wide || !(square < kLargeQuery);
            // (a NaN is not bounded; a wave by itself: the barriers are the same)
            // (and a wave without rows only stages)
            bounded = __builtin_amdgcn_ballot_w64(!(norm * bound(square) <= kBound) || a.m != 0.f || (DENSE && members == 0)) == 0;
        }
        count = __builtin_amdgcn_readfirstlane(count);
        // Tile t is part t % sub of block t / sub; only the sequence's last one may be short.
        const int shift = p.bs == 64 ? 0 : p.bs == 128 ? 1 : 2, sub = 1 << shift;
        const int rest = end - __builtin_amdgcn_readlane(block, count - 1) * p.bs;   // keys from the last block on
        const int total = ((count - 1) << shift) + min(sub, (rest + 63) / 64), whole = ((count - 1) << shift) + min(sub, rest / 64);
        auto fetch = [&](int t, Staged& to) {
            t = min(t, total - 1);
            load(__builtin_amdgcn_readlane(block, t >> shift), t & (sub - 1), to);
        };
        uint32_t of;
        bool member;
        Factors ft;
        auto meet = [&](int i) {
            auto lane_f = [&](float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), i)); };
            of = (uint32_t)__builtin_amdgcn_readlane(members, i);
            ft = Factors{lane_f(f.ck), lane_f(f.lv), lane_f(f.iv)};
            member = DENSE || row.in(of);   // (rows that do not exist are not stored)
        };
        int t = 0;
        // (past the last tile the staged one is put and loaded once more, to no effect: no branch in the way)
        // Tiles on their way to registers: two where the accumulators leave room for them
        constexpr int kAhead = DENSE && !SAFE ? 2 : 1;
        Staged ahead[kAhead];
        auto stage = [&](Staged& x) {
            put(~t & 1, x);
            __builtin_amdgcn_sched_barrier(0);   // (x is free before it is loaded again)
            fetch(t + 1 + kAhead, x);
        };
        put(0, r);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) fetch(1 + i, ahead[i]);
        // Two loops, each with one way through, so that the accumulators stay where they are
        auto whole_tile = [&](Staged& x) {
            lds_barrier();
            meet(t >> shift);
            a.has = a.has || member;
            if constexpr (DENSE) attend_whole(L.tile[t & 1], qf, member, ft, a, [&] { stage(x); });
            else {
                if (of != 0) attend_whole(L.tile[t & 1], qf, member, ft, a, [] {});
                stage(x);
            }
            ++t;
        };
        auto any_tile = [&](Staged& x) {
            lds_barrier();
            meet(t >> shift);
            stage(x);
            if (of != 0) attend_tile<SAFE>(L.tile[t & 1], qf, member, t < whole ? 64 : rest & 63, ft, a);
            ++t;
        };
        if (bounded) {
            if constexpr (kAhead == 1)
                while (t < whole) whole_tile(ahead[0]);
            else {
                while (t + 1 < whole) {
                    whole_tile(ahead[0]);
                    whole_tile(ahead[1]);
                }
                if (t < whole) {
                    whole_tile(ahead[0]);
                    ahead[0] = ahead[1];   // (for the last tile, if it is short)
                }
            }
        }
        if constexpr (kAhead == 1)
            while (t < total) any_tile(ahead[0]);
        else
            while (t < total) {
                any_tile(ahead[0]);
                if (t < total) any_tile(ahead[1]);
            }
        lds_barrier();   // the buffers are free for the next blocks
    }
};

template <bool FP8, bool DENSE, bool SAFE, int WAVES, typename Lds>
__device__ __forceinline__ void attend(const CacheAttnParams& p, Lds& L, int b, int h, int n0, int split, int splits, const Row& row, int wave_live,
                                       float w, AttnState& a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    a.o[0] = a.o[1] = splat(0.f);
    a.m = a.l = 0.f;
    a.has = a.wide = false;
    const int end = seq_keys(p, b);
    bf16x8 qf[4];   // step ds: dims 32 (ds / 2) + 16 hh + 8 (ds % 2) .. (see qcache.h)
    auto load_q = [&] {
        const bf16_t* qr = p.q + b * p.q_sb + row.n * p.q_sn + row.head * p.q_sh + 16 * (lane >> 5);
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) qf[ds] = as_bf16x8(ld16(qr + 32 * (ds >> 1) + 8 * (ds & 1)));
        if constexpr (SAFE) {
            bool large = false;
#pragma unroll
            for (int ds = 0; ds < 4; ++ds) large = large || large_query(qf[ds]);
            large = __builtin_amdgcn_ballot_w64(large) >> (lane & 31) & 0x100000001ull;   // (either half of the row)
            a.c = row_factor(p.c, large);
#pragma unroll
            for (int ds = 0; ds < 4; ++ds) qf[ds] = within(qf[ds], large);
        }
    };
    Walk<FP8, DENSE, SAFE, WAVES, Lds> walk{p, L, b, h, end, w, qf, row, a};
    const int live = (int)(((int64_t)end + p.bs - 1) / p.bs);   // blocks with a key
    if constexpr (DENSE) {
        load_q();
        const int first = share_begin(live, split, splits), past = share_begin(live, split + 1, splits);
        for (int e0 = first; e0 < past; e0 += 64) walk.blocks(min(64, past - e0), min(e0 + lane, past - 1), wave_live);
    } else {
        load_q();
        const bool by_block = p.keys != nullptr;
        for (int c0 = 0; c0 < live; c0 += kUnion) {
            const int found = unite(p, L, b, h, n0, end, c0, min(kUnion, live - c0), split, by_block ? splits : 1);
            const int first = by_block ? 0 : (int)((uint32_t)(found * split) / (uint32_t)splits);
            const int past = by_block ? found : (int)((uint32_t)(found * (split + 1)) / (uint32_t)splits);
            for (int e0 = first; e0 < past; e0 += 64) {
                const int count = min(64, past - e0), u = L.list[e0 + min(lane, count - 1)];
                walk.blocks(count, c0 + u, (int)L.members[u][wave]);
            }
            __syncthreads();
        }
    }
}

// A part's sum of weights 2^m l in joins: no weight overflows, whatever m and l are, and parts of one m weigh as their l,
// also where m's unit is more than the exponent of l (which therefore stays beside m, not in it).
struct Sum {
    float m, y;   // l = 2^e y
    int e;
    __device__ __forceinline__ explicit Sum(float2 ml) : m(ml.x), y(__builtin_amdgcn_frexp_mantf(ml.y)), e(__builtin_amdgcn_frexp_expf(ml.y)) {}
    __device__ __forceinline__ float top() const { return y == 0.f ? -INFINITY : m + (float)e; }   // (l = 0: no key)
    // relative to the largest top
    __device__ __forceinline__ float weight(float most) const { return y == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - most + (float)e) * y; }
};

// The result of a row, or its part of it
__device__ __forceinline__ void put_row(const CacheAttnParams& p, const Row& row, int64_t part, int split, int splits, float w, AttnState& a) {
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const float l = xor32_add(a.l), f = l == 0.f ? 0.f : 1.f / l;   // (a row without a key, or with none above -inf: zeros)
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) a.o[dt] *= f;   // (before w: 1 / l and w need not fit together)
    if (splits == 1) {
        store_row(p.out, row.at, lane, a.o, w);
        return;
    }
    float* d = p.part_o + (split * p.parts + part) * 64 + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<float4*>(d + 32 * dt + 8 * g4) =
                make_float4(a.o[dt][4 * g4] * w, a.o[dt][4 * g4 + 1] * w, a.o[dt][4 * g4 + 2] * w, a.o[dt][4 * g4 + 3] * w);
    if (hh == 0) p.part_ml[split * p.parts + part] = make_float2(a.m, l);
}

template <bool FP8, bool DENSE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 3) void cache_attn_kernel(CacheAttnParams p) {
    static_assert(DENSE || WAVES == kWaves, "the union's members are those of four waves");
    __shared__ std::conditional_t<DENSE, DenseLds, SetsLds> L;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // whole tiles of rows, then the others, each with its keys in shares
    int split = 0, splits = 1, tile = blockIdx.x;
    if ((int)blockIdx.x < p.whole) tile = xcd_runs(blockIdx.x, p.whole);
    else {
        const int i = blockIdx.x - p.whole;
        splits = p.splits;
        tile = p.whole + i / splits;
        split = i % splits;
    }
    const int tile_id = tile % p.qtiles, rest = tile / p.qtiles, h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * WAVES * p.QW;
    if constexpr (!DENSE) load_tokens(p, L, b, h, n0);
    // (formed anew where it is needed again: the loops between have no register for it)
    auto my_row = [&] {
        int first = n0;
        asm volatile("" : "+s"(first));
        Row row;
        if constexpr (DENSE) row.init(p, [&](int i) { return min(first + i, p.Nq - 1); }, b, h, first, wave, lane & 31);
        else row.init(p, [&](int i) { return L.tokens[i]; }, b, h, first, wave, lane & 31);
        return row;
    };
    auto put = [&](AttnState& a, float w, bool ok) {
        const Row row = my_row();
        const int64_t part = (int64_t)(tile - p.whole) * (WAVES * kRows) + wave * kRows + (lane & 31);
        if (splits > 1 && split == 0 && hh == 0) p.part_at[part] = row.live ? row.at : -1;
        if (row.live && ok) put_row(p, row, part, split, splits, w, a);
    };
    const float w = value_unit(p.cache, b, h);
    AttnState a;
    bool ok;
    {
        const Row row = my_row();
        const int wave_live = __builtin_amdgcn_ballot_w64(row.live) ? -1 : 0;   // (a wave without rows only stages)
        attend<FP8, DENSE, false, WAVES>(p, L, b, h, n0, split, splits, row, wave_live, w, a);
        const bool fine = finite(a.o[0]) && finite(a.o[1]) && a.l - a.l == 0.f && !a.wide && fabsf(a.m) <= kFar;
        const int other = __shfl_xor((int)fine, 32);   // (the other half of the row)
        ok = !row.live || (fine && other);
    }
    put(a, w, ok);
    if (!__syncthreads_or(!ok)) return;
    const Row row = my_row();
    attend<FP8, DENSE, true, WAVES>(p, L, b, h, n0, split, splits, row, __builtin_amdgcn_ballot_w64(row.live) ? -1 : 0, 1.f, a);
    put(a, 1.f, !ok);
}

// ------------------------------------------------------------------ few rows

// One token above all: no more than 16 rows (token, head) of a kv head.  A workgroup's waves take the tiles
// of 64 keys of its share in turn, straight from memory into the operands of v_mfma_f32_16x16x32_bf16
// (lane group g = lane / 16): in step m the keys' rows 4 g + i are tokens 16 g + 4 m + i, so that a lane
// ends with the scores of the 16 tokens that its chunk of the values holds.  A tile is requested while
// the one before is computed (two ahead need 196 registers: 32 us for 21 over 196608 keys).
// Eight waves where one workgroup takes a head's keys: a wave alone issues a vector instruction in four cycles, about
// 1 us a tile, and two of a SIMD hide each other's waits (one token, 16 blocks of 128, a call: 14.4 us,
// of 4 waves 16.1, of 16 waves 15.5; 13.7 since the shares and the join became shorter).
constexpr int kFewRows = 16, kFewEntries = 64;

struct FewState {
    f32x4 o[4];       // O^T [16 dims]: dims 16 dg + 4 g + i
    float m, l;
    bool has, wide;   // as AttnState's
};
struct Codes { uint4 k[4], v[4]; float ks, vs; };

__device__ __forceinline__ float xor16_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_add(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <bool FP8>
__device__ __forceinline__ bf16x8 codes8(uint32_t a, uint32_t b) {
    const uint2 x = codes_bf16<FP8>(a), y = codes_bf16<FP8>(b);
    return as_bf16x8(make_uint4(x.x, x.y, y.x, y.y));
}

template <bool FP8, bool SAFE>
__device__ __forceinline__ void attend_few(const Codes& t, const bf16x8 (&qf)[2], bool member, int valid, float c, float w, FewState& a) {
    const int g = (threadIdx.x & 63) >> 4;
    bool wide;
    const Factors f = factors<SAFE>(c, t.ks, t.vs, w, wide);
    a.wide = a.wide || (wide && member);
    f32x4 s[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        s[m] = mfma16(codes8<FP8>(t.k[m].x, t.k[m].y), qf[0], f32x4{0.f, 0.f, 0.f, 0.f});
        s[m] = mfma16(codes8<FP8>(t.k[m].z, t.k[m].w), qf[1], s[m]);
    }
    if (valid < 64) {
        seldom();
        int left = valid - 16 * g;
        asm volatile("" : "+v"(left));
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][i] = 4 * m + i < left ? s[m][i] : -INFINITY;
    }
    float mt = s[0][0];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = __builtin_elementwise_maximum(mt, s[m][i]);
    const float ck = SAFE ? score_factor(c, f.ck) : f.ck;
    mt = xor32_max(xor16_max(mt)) * ck;
    const bool some = member && mt > -INFINITY, move = some && (!a.has || mt > a.m + (SAFE ? 0.f : kTau));
    if (__builtin_amdgcn_ballot_w64(move)) {
        const float alpha = move && a.has ? __builtin_amdgcn_exp2f(a.m - mt) : 1.f;
        a.m = move ? mt : a.m;
#pragma unroll
        for (int dg = 0; dg < 4; ++dg) a.o[dg] *= alpha;
        a.l *= alpha;
    }
    a.has = a.has || some;
    const float ref = member ? (SAFE ? f.iv : f.lv) - a.m : -INFINITY;   // P = 0 for the others
    auto weight = [&](float x) { return __builtin_amdgcn_exp2f(SAFE ? times_plus(x, ck, ref) : fmaf(x, ck, ref)); };
    // P in two terms, 16 bits of it: the products wait for the codes, and a single row does not average the rounding
    bf16x8 pb[2], rest[2];
    float lt = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t u[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = weight(s[2 * j + (i >> 1)][2 * (i & 1)]), x1 = weight(s[2 * j + (i >> 1)][2 * (i & 1) + 1]);
            lt += x0 + x1;
            u[i] = pack_bf16x2(x0, x1);
            y[i] = pack_bf16x2(x0 - bf_lo(u[i]), x1 - bf_hi(u[i]));
        }
        pb[j] = as_bf16x8(make_uint4(u[0], u[1], u[2], u[3]));
        rest[j] = as_bf16x8(make_uint4(y[0], y[1], y[2], y[3]));
    }
    if constexpr (SAFE) {
        if (member) a.l += lt;
    } else a.l = fmaf(lt, f.iv, a.l);
#pragma unroll
    for (int dg = 0; dg < 4; ++dg) {
        const bf16x8 v0 = codes8<FP8>(t.v[dg].x, t.v[dg].y), v1 = codes8<FP8>(t.v[dg].z, t.v[dg].w);
        auto product = [&](f32x4 y) { return mfma16(v1, pb[1], mfma16(v0, pb[0], mfma16(v1, rest[1], mfma16(v0, rest[0], y)))); };
        if constexpr (SAFE) {
            const f32x4 y = product(f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) a.o[dg][i] = member ? fmaf(y[i], f.lv, a.o[dg][i]) : a.o[dg][i];
        } else a.o[dg] = product(a.o[dg]);
    }
}

template <bool FP8, bool DENSE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 ? 3 : 1) void cache_attn_few_kernel(CacheAttnParams p) {
    __shared__ __attribute__((aligned(16))) float O[WAVES][kFewRows][64];
    __shared__ float2 ml[WAVES][kFewRows];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits, h = rest % p.Hk, b = rest / p.Hk;
    const int end = seq_keys(p, b), shift = p.bs == 64 ? 6 : p.bs == 128 ? 7 : 8, sub = 1 << (shift - 6), rows = p.Nq * p.G;   // bs = 2^shift
    const bool row_live = r < rows;
    const int token = row_live ? r / p.G : 0, head = h * p.G + (row_live ? r - token * p.G : 0);
    const bf16_t* qr = p.q + b * p.q_sb + token * p.q_sn + head * p.q_sh + 16 * g;
    bf16x8 qf[2] = {as_bf16x8(ld16(qr)), as_bf16x8(ld16(qr + 8))};
    // the call's blocks: all of them, or those that the tokens' entries name, one in a lane of every wave
    int units, blk = -1, rank = 0;
    uint32_t tokens = 0;
    bool lead = false;
    if constexpr (DENSE) units = (int)(((int64_t)end + 63) / 64);
    else {
        const int entries = p.Nq * p.K;
        if (lane < entries) {
            const int t = lane / p.K;
            const int64_t u = p.idx[(((int64_t)b * p.Nq + t) * p.Hk + h) * p.K + lane - t * p.K];
            blk = u >= 0 && u < p.nb && u * p.bs < end ? (int)u : -1;
        }
        lead = blk >= 0;
        for (int j = 0, t = 0, of = 0; j < entries; ++j) {
            const bool same = __builtin_amdgcn_readlane(blk, j) == blk;
            tokens |= same ? 1u << t : 0u;
            lead = lead && !(same && j < lane);
            if (++of == p.K) {
                of = 0;
                ++t;
            }
        }
        const uint64_t leads = __builtin_amdgcn_ballot_w64(lead);
        rank = (int)__builtin_popcountll(leads & ((1ull << lane) - 1ull));
        units = (int)__builtin_popcountll(leads) * sub;
    }
    const int first = share_begin(units, split, p.splits), past = share_begin(units, split + 1, p.splits);
    const int kt = r >> 3, ko = kt * 2048 + (g >> 1) * 1024 + (g & 1) * 512 + (r & 7) * 16;
    const int vo = (g >> 1) * 2048 + (g & 1) * 512 + r * 16;
    // unit u: its first key, and the tokens that have it
    auto where = [&](int u, uint32_t& of) {
        of = ~0u;
        if constexpr (DENSE) return u * 64;
        else {
            const int which = u >> (shift - 6);
            const int src = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(lead && rank == which));
            of = (uint32_t)__builtin_amdgcn_readlane((int)tokens, src);
            return __builtin_amdgcn_readlane(blk, src) * p.bs + (u - which * sub) * 64;
        }
    };
    auto load = [&](int key0, Codes& t) {
        const int j = key0 >> shift;
        const int64_t at = block_at(p.cache, b, j, h), from = (at << (shift + 6)) + (key0 - (j << shift)) * 64;
        const uint8_t* kc = static_cast<const uint8_t*>(p.cache.k_codes) + from;
        const uint8_t* vc = static_cast<const uint8_t*>(p.cache.v_codes) + from;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            t.k[i] = ld16(kc + ko + 128 * i);
            t.v[i] = ld16(vc + vo + (i >> 1) * 1024 + (i & 1) * 256);
        }
        t.ks = p.cache.k_scale[at];
        t.vs = p.cache.v_scale[at];
    };
    FewState a;
    float w = value_unit(p.cache, b, h), c = p.c;
    auto walk = [&](auto safe) {
#pragma unroll
        for (int dg = 0; dg < 4; ++dg) a.o[dg] = f32x4{0.f, 0.f, 0.f, 0.f};
        a.m = a.l = 0.f;
        a.has = a.wide = false;
        if (first + wave >= past) return;
        Codes next;
        uint32_t of_next;
        int key_next = where(first + wave, of_next);
        load(min(key_next, end - 1), next);   // (a block's later tiles may lie behind the end)
        for (int u = first + wave; u < past; u += WAVES) {
            const Codes t = next;
            const uint32_t of = of_next;
            const int key0 = key_next;
            if (u + WAVES < past) {
                key_next = where(u + WAVES, of_next);
                load(min(key_next, end - 1), next);
            }
            if (key0 < end)
                attend_few<FP8, decltype(safe)::value>(t, qf, row_live && (DENSE || (of >> token & 1)), min(64, end - key0), c, w, a);
        }
    };
    walk(std::false_type{});
    bool large = large_query(qf[0]) || large_query(qf[1]);
    bool ok = !a.wide && !large && a.l - a.l == 0.f && fabsf(a.m) <= kFar;
#pragma unroll
    for (int dg = 0; dg < 4; ++dg)
#pragma unroll
        for (int i = 0; i < 4; ++i) ok = ok && a.o[dg][i] - a.o[dg][i] == 0.f;
    if (__builtin_amdgcn_ballot_w64(!ok)) {   // (a wave by itself, with all of its rows)
        w = 1.f;
        large = __builtin_amdgcn_ballot_w64(large) >> r & 0x1000100010001ull;   // (any part of the row)
        c = row_factor(p.c, large);
#pragma unroll
        for (int i = 0; i < 2; ++i) qf[i] = within(qf[i], large);
        walk(std::true_type{});
    }
    const float l = xor32_add(xor16_add(a.l)), f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int dg = 0; dg < 4; ++dg)
        *reinterpret_cast<float4*>(&O[wave][r][(16 * dg + 4 * g) ^ (4 * r)]) =
            make_float4(a.o[dg][0] * f * w, a.o[dg][1] * f * w, a.o[dg][2] * f * w, a.o[dg][3] * f * w);
    if (g == 0) ml[wave][r] = make_float2(a.m, l);
    __syncthreads();
    // 16 threads a row
    const int row = tid / 16, d = 4 * (tid % 16);
    if (row >= rows) return;
    float2 part[WAVES];
    float4 x[WAVES];
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        part[i] = ml[i][row];
        x[i] = *reinterpret_cast<const float4*>(&O[i][row][d ^ (4 * row)]);
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, Sum(part[i]).top());
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const float y = Sum(part[i]).weight(m);
        sum += y;
        o.x = fmaf(y, x[i].x, o.x); o.y = fmaf(y, x[i].y, o.y); o.z = fmaf(y, x[i].z, o.z); o.w = fmaf(y, x[i].w, o.w);
    }
    const float y = sum == 0.f ? 0.f : 1.f / sum;
    const int t = row / p.G;
    const int64_t at = ((int64_t)b * p.Nq + t) * p.Hq + h * p.G + row - t * p.G;
    if (p.splits == 1) {
        *reinterpret_cast<uint2*>(p.out + at * 64 + d) = make_uint2(pack_bf16x2(o.x * y, o.y * y), pack_bf16x2(o.z * y, o.w * y));
        return;
    }
    *reinterpret_cast<float4*>(p.part_o + (split * p.parts + at) * 64 + d) = make_float4(o.x * y, o.y * y, o.z * y, o.w * y);
    if (d == 0) p.part_ml[split * p.parts + at] = make_float2(m, sum);
}

// ------------------------------------------------------------------ joins

// Joins the splits' partials: 16 lanes a row, 4 dims each, and TEAM such groups a row that take its splits in
// turn, up to 16 each: one for up to 16 splits, 16 for up to 64, 64 (a workgroup of 1024 threads) for more.  A
// lane holds the weight of one split, and the first of the partials are on their way before the weights are known.
constexpr int kJoinMost = 1024;
template <int TEAM>
__global__ __launch_bounds__(TEAM == 64 ? 1024 : kThreads) void cache_attn_join_kernel(CacheAttnParams p) {
    constexpr int kGroups = TEAM == 64 ? 64 : kThreads / 16, kAhead = 4;
    __shared__ float4 part[TEAM == 1 ? 1 : kGroups][16];
    __shared__ float most[kGroups], sums[kGroups];
    const int group = threadIdx.x / 16, j = threadIdx.x % 16, d = 4 * j, of = group % TEAM;
    const int64_t rows = p.parts, mine = (int64_t)blockIdx.x * (kGroups / TEAM) + group / TEAM, row = mine < rows ? mine : rows - 1;
    const int64_t at = p.part_at != nullptr ? p.part_at[row] : row;
    if (TEAM > 1 && at < 0) return;   // (all of a workgroup: no such row)
    const int n = of < p.splits ? (p.splits - of + TEAM - 1) / TEAM : 0;   // splits of the group: of + TEAM i
    auto o_of = [&](int i) { return *reinterpret_cast<const float4*>(p.part_o + ((of + TEAM * i) * rows + row) * 64 + d); };
    const float2 ml = j < n ? p.part_ml[(of + TEAM * j) * rows + row] : make_float2(0.f, 0.f);
    float4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = n > 0 ? o_of(min(i, n - 1)) : make_float4(0.f, 0.f, 0.f, 0.f);
    const Sum share(ml);
    float m = share.top();
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    if constexpr (TEAM > 1) {
        if (j == 0) most[group] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TEAM; i += 16) m = fmaxf(m, most[group / TEAM * TEAM + i + j]);
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    }
    const float w = share.weight(m);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int i, const float4& y) {
        const float f = __shfl(w, (threadIdx.x & 48) + i);
        l += f;
        o.x = fmaf(f, y.x, o.x); o.y = fmaf(f, y.y, o.y); o.z = fmaf(f, y.z, o.z); o.w = fmaf(f, y.w, o.w);
    };
    // (16 steps in all groups of a wave, so that every lane is there for the exchange; beyond n weights are 0)
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(i, ahead[i]);
    for (int i = kAhead; i < (p.splits + TEAM - 1) / TEAM; ++i) add(i, n > 0 ? o_of(min(i, n - 1)) : make_float4(0.f, 0.f, 0.f, 0.f));
    if constexpr (TEAM > 1) {
        part[group][j] = o;
        if (j == 0) sums[group] = l;
        __syncthreads();
        if (of != 0) return;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
#pragma unroll 16
        for (int i = 0; i < TEAM; ++i) {
            const float4 y = part[group + i][j];
            l += sums[group + i];
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
    }
    if (mine >= rows || at < 0) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + at * 64 + d) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
}

// ------------------------------------------------------------------ host

// Shares of the keys of few rows: four workgroups a CU, where a row has no more than kFewShares then, and else one a
// CU: its join is the longer (one point over 196608 keys, 75 MB in e4m3: 20.5 us in 85 shares of each head, 23.3 in
// 170 and in 341; 24 tracks of 16 heads, 113 MB in int8: 25 us in 10 shares, 29 in 2).  One share and no join up to
// kFewWhole tiles (2048 keys: 13 us, 17 in four shares), and no fewer than kFewTiles in a share, two a wave (4096 keys:
// 16 us in eight shares, 17 in two, 21 in one).
constexpr int64_t kFewGroups = 1024, kFewShares = 64, kFewWhole = 40, kFewTiles = 8;
constexpr int kManyWaves = 8;   // of a workgroup that takes all keys of a head of few rows
static_assert(kJoinMost >= kFewGroups, "the join takes every share");
// A dense call's layout is the one of the least time by these, in microseconds: a tile of 64 keys of a chip full of
// rows, in workgroups of 4 waves, three a CU, or of 12, one a CU, which convert a tile once for 384 rows; a join, and a
// row's part of it.  (12 heads on 3 over 49152 keys, 4 | 12 waves | the choice: 128 tokens 44 | 46 | 44 us, 1000 tokens
// 192 | 183 | 182, 12288 tokens 1875 | 1660 | 1660; 6000 tokens, whose last round is
// nearly empty, 1021 without shares of it, 850 with; 12288 tokens over 12288 keys of 4 members 1845 | 1677 | 1677.)
constexpr double kTile = 1.7, kWideTile = 1.45, kJoinTime = 4., kPartTime = 6e-5;

// Whether the call is one of cache_attn_few_kernel
bool few(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    const int64_t rows = (int64_t)nq * (hq / c.num_kv_heads);
    return rows <= kFewRows && (int64_t)nq * K <= kFewEntries;
}

// Whether the tokens' order is looked for: its two launches cost 7 us and more, and unions of tokens in no order cost
// less up to about 8192 entries of all heads (scattered tokens, 3 kv heads: 40 of 16 blocks 24 us, 31 with the launches;
// 500 of 4 blocks 30 and 35; 200 of 16 blocks, 9600 entries, 37 and 37; 500 of 16 blocks 54 and 37).
bool ordered(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    return K > 0 && !few(c, nq, hq, K) && (double)c.num_kv_heads * c.batch * nq * K > 8192.;
}

template <int WAVES>
const void* few_kernel(bool fp8, bool sets) {
    return fp8 ? (sets ? (const void*)&cache_attn_few_kernel<true, false, WAVES> : (const void*)&cache_attn_few_kernel<true, true, WAVES>)
               : (sets ? (const void*)&cache_attn_few_kernel<false, false, WAVES> : (const void*)&cache_attn_few_kernel<false, true, WAVES>);
}

// How a call is laid out: waves of a workgroup, tiles of rows, those taken whole, and shares of the others' keys.
struct Plan {
    int waves;
    int64_t qtiles, tiles, whole, splits, parts;   // tiles of a (member, kv head), and of all; rows that are joined
    size_t part_o, part_ml, part_at, bytes;        // places in the workspace, and what the partials take of it; then
    size_t order;                                  // bytes of the tokens' order (0: they stay in their own)
    int64_t groups() const { return whole + (tiles - whole) * splits; }
};
Plan plan_of(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    Plan a{};
    a.waves = kWaves;
    const int G = hq / c.num_kv_heads;
    const int64_t heads = (int64_t)c.num_kv_heads * c.batch, sub = c.block_size / 64;
    if (few(c, nq, hq, K)) {
        const int64_t tiles = K > 0 ? nq * K * sub : c.num_blocks * sub;
        a.tiles = heads;
        a.splits = kFewGroups / heads;
        if (a.splits > kFewShares) a.splits = std::max(kFewShares, 256 / heads);
        a.splits = tiles <= kFewWhole ? 1 : std::max<int64_t>(1, std::min(a.splits, tiles / kFewTiles));
        if (a.splits == 1 && tiles > kWaves) a.waves = kManyWaves;
        a.parts = (int64_t)c.batch * nq * hq;
    } else if (K > 0) {
        // Shares where there are few tiles: of a union that may be as many blocks as the tile's tokens have entries, three
        // workgroups a CU, two where the join is one of teams (16 blocks of 64 a token: 17 scattered tokens 17 us,
        // 26 in 16 shares; 40, their order looked for, 32 and 41 in 16; 200 33 and 35 in 36; 1000 39 and 73 in one; 3500 57
        // in one or two)
        const int64_t per = kWaves * (kRows / G), tokens = std::min<int64_t>(nq, per);
        a.qtiles = (nq + per - 1) / per;
        a.tiles = a.qtiles * heads;
        a.splits = a.tiles >= 256 ? 1 : std::min<int64_t>({768 / a.tiles, std::max<int64_t>(16, 512 / a.tiles), tokens * K, 64});
        a.whole = a.splits == 1 ? a.tiles : 0;
        a.parts = (a.tiles - a.whole) * kWaves * kRows;
    } else {   // full rounds of the chip, and the rest's keys in shares
        double best = INFINITY;
        for (int waves : {4, 12}) {
            const int64_t per = waves * (kRows / G), qtiles = (nq + per - 1) / per, tiles = qtiles * heads, slots = waves == 4 ? 768 : 256;
            const int64_t whole = tiles / slots * slots, rest = tiles - whole;
            const double round = c.num_blocks * sub * (waves == 4 ? kTile : kWideTile);
            auto take = [&](int64_t unsplit, int64_t splits) {
                const int64_t groups = (tiles - unsplit) * splits, left = groups % slots, parts = splits > 1 ? rest * waves * kRows : 0;
                // (a last round of one or two workgroups a CU takes less time than one of three)
                const double rounds = groups / slots + (left == 0 ? 0. : waves == 12 || left > 512 ? 1. : left > 256 ? .75 : .5);
                const double time = (unsplit / slots + rounds / splits) * round + (splits > 1 ? kJoinTime + splits * parts * kPartTime : 0.);
                if (time >= best) return;
                best = time;
                a.waves = waves; a.qtiles = qtiles; a.tiles = tiles; a.whole = unsplit; a.splits = splits; a.parts = parts;
            };
            take(0, 1);
            if (rest > 0)
                for (int64_t fill : {256, 512, 768, 1024, 1536, 2304}) {
                    const int64_t splits = std::min<int64_t>({fill / rest, std::max<int64_t>(1, c.num_blocks / 4), kJoinMost});
                    if (splits > 1) take(whole, splits);
                }
        }
        if (a.splits == 1) a.whole = a.tiles;
    }
    if (a.splits > 1) {
        a.part_ml = up(a.splits * a.parts * kHeadDim * sizeof(float));
        a.part_at = a.part_ml + up(a.splits * a.parts * sizeof(float2));
        a.bytes = a.part_at + up(a.parts * sizeof(int64_t));
    }
    return a;
}

// A call's checks that need no pointer, and its plan
int plan_call(const mosaic_kv_cache* cache, int32_t nq, int32_t hq, int32_t d, int32_t K, Plan& plan) {
    if (int e = check_cache(cache)) return e;
    if (nq <= 0) return MOSAIC_ERR_SHAPE;
    if (d != kHeadDim) return MOSAIC_ERR_HEAD_DIM;
    const int hk = cache->num_kv_heads;
    if (hq <= 0 || hq % hk) return MOSAIC_ERR_HEADS;
    if (hq / hk > 16 || K > kMaxSelected) return MOSAIC_ERR_UNSUPPORTED;
    if (K < 0) return MOSAIC_ERR_BLOCK_COUNT;
    if (nq > 0x7fffffff - 1024) return MOSAIC_ERR_SHAPE;   // (tokens past the last stay in 31 bits)
    plan = plan_of(*cache, nq, hq, K);
    if (!grid_fits(plan.groups(), 64 * plan.waves)) return MOSAIC_ERR_SHAPE;
    plan.order = ordered(*cache, nq, hq, K) ? order_bytes(cache->batch, nq, hq, hk) : 0;
    const int64_t heads = (int64_t)cache->batch * hk;
    if (plan.order > 0 && (!grid_fits(heads * key_chunks(nq), kThreads) || !grid_fits(heads, kOrderThreads))) return MOSAIC_ERR_SHAPE;
    return MOSAIC_OK;
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

size_t mosaic_cache_attn_fwd_workspace_size(const mosaic_kv_cache* cache, int32_t num_queries, int32_t num_q_heads, int32_t block_count) {
    Plan plan;
    if (plan_call(cache, num_queries, num_q_heads, kHeadDim, block_count, plan) != MOSAIC_OK) return 0;
    return plan.bytes + plan.order;
}

int mosaic_cache_attn_fwd(mosaic_bnhd q, const mosaic_kv_cache* cache, const int64_t* block_indices, const int32_t* kv_lens,
                          int32_t num_queries, int32_t num_q_heads, int32_t head_dim, int32_t block_count, float softmax_scale,
                          void* out, void* workspace, size_t workspace_bytes, void* stream) {
    Plan plan;
    if (int e = plan_call(cache, num_queries, num_q_heads, head_dim, block_count, plan)) return e;
    if (!scale_ok(softmax_scale)) return MOSAIC_ERR_UNSUPPORTED;
    if (q.ptr == nullptr || out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if ((block_indices == nullptr) != (block_count == 0)) return MOSAIC_ERR_BLOCK_COUNT;
    if (!aligned(q.ptr, 16) || q.stride_b % 8 || q.stride_n % 8 || q.stride_h % 8) return MOSAIC_ERR_ALIGNMENT;
    if (!aligned(block_indices, 8) || !aligned(out, 16) || !aligned(kv_lens, 4)) return MOSAIC_ERR_ALIGNMENT;
    const size_t need = plan.bytes + plan.order;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256))) return MOSAIC_ERR_WORKSPACE;
    CacheAttnParams p{};
    p.cache = *cache;
    p.q = static_cast<const bf16_t*>(q.ptr); p.q_sb = q.stride_b; p.q_sn = q.stride_n; p.q_sh = q.stride_h;
    p.idx = block_indices; p.lens = kv_lens;
    p.B = cache->batch; p.Nq = num_queries; p.Nk = cache->capacity; p.Hq = num_q_heads; p.Hk = cache->num_kv_heads;
    p.G = p.Hq / p.Hk; p.QW = kRows / p.G; p.bs = cache->block_size; p.K = block_count; p.nb = cache->num_blocks;
    p.qw_inverse = (65536 + p.QW - 1) / p.QW;
    p.qtiles = (int)plan.qtiles; p.splits = (int)plan.splits; p.whole = (int)plan.whole; p.parts = plan.parts;
    p.out = static_cast<bf16_t*>(out);
    p.c = (softmax_scale > 0.f ? softmax_scale : 0.125f) * kLog2e;
    char* ws = static_cast<char*>(workspace);
    const bool small = few(*cache, num_queries, num_q_heads, block_count);
    if (p.splits > 1) {
        p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
        p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
        if (!small) p.part_at = reinterpret_cast<int64_t*>(ws + plan.part_at);
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (plan.order > 0) {
        place_order(p, ws + plan.bytes);
        if (int e = launch_order(p, s)) return e;
    }
    void* args[] = {&p};
    const bool fp8 = cache->code_type == MOSAIC_CODE_E4M3, sets = block_count > 0;
    const void* fn;
    if (small && plan.waves == kManyWaves) fn = few_kernel<kManyWaves>(fp8, sets);
    else if (small) fn = few_kernel<kWaves>(fp8, sets);
    else if (sets) fn = fp8 ? (const void*)&cache_attn_kernel<true, false, 4> : (const void*)&cache_attn_kernel<false, false, 4>;
    else if (plan.waves == 12) fn = fp8 ? (const void*)&cache_attn_kernel<true, true, 12> : (const void*)&cache_attn_kernel<false, true, 12>;
    else fn = fp8 ? (const void*)&cache_attn_kernel<true, true, 4> : (const void*)&cache_attn_kernel<false, true, 4>;
    if (launch(fn, dim3((unsigned)plan.groups()), args, s, 64 * plan.waves) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (p.splits == 1) return MOSAIC_OK;
    void* jargs[] = {&p};
    const int team = p.splits <= 16 ? 1 : p.splits <= 64 ? 16 : 64;
    const void* join = team == 1    ? (const void*)&cache_attn_join_kernel<1>
                       : team == 16 ? (const void*)&cache_attn_join_kernel<16>
                                    : (const void*)&cache_attn_join_kernel<64>;
    const unsigned joins = (unsigned)(team == 1 ? (p.parts + 15) / 16 : p.parts);
    return launch(join, dim3(joins), jargs, s, team == 64 ? 1024 : kThreads) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
