// cattn.hip -- attention of query tokens over a key/value cache held in 8 bits (gfx950).
//
// Row (b, n, g) = query token n and query head g of kv head h; over its keys u, those below the
// sequence's length and, where the call names key blocks, of the token's blocks:
//   o = sum_u p_u v_u / sum_u p_u,  p_u = exp2(c q.k_u - m),  c = softmax_scale log2 e,
//   k_u = ks code, v_u = vs code, ks and vs the scales of u's block and head
// Codes are whole numbers of at most 8 bits or e4m3, exact in bf16, so the products are of bf16 operands
// without a rounding of theirs.  ks goes into the factor of the scores and vs into the exponent,
//   P = exp2(c ks q.code_k + log2(vs / w) - m),  O = sum P code_v,  l = sum P w / vs,  o = w O / l,
// so that neither costs an instruction per score (w: a scale that a workgroup takes first).  fp32 scores,
// maxima, sums and accumulators; P is rounded to bf16 for the product with the values (half a step of
// bf16 per term, as the output's own rounding), and l sums the rounded P.
//
// A workgroup takes 4 waves x QW = 32 / G tokens of one kv head, a wave the 32 rows (token, head) of
// its tokens; the codes of 64 keys are converted once, by all four waves, into operand order in LDS.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

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
    float* part_o;             // [splits, rows, 64] (splits > 1): o of a split's keys
    float2* part_ml;           // [splits, rows] (m, l): 2^m l is the sum of its weights, l in [1, 2), or 0
    float c;
};

// A tile of 64 keys in operand order: keys [kt 2][step 4][lane 64][8], values [kt 2][dt 2][step 2][lane 64][8]
struct CacheTile {
    __attribute__((aligned(1024))) bf16_t K[64 * 64];
    __attribute__((aligned(1024))) bf16_t V[64 * 64];
};
struct DenseLds { CacheTile tile[2]; };
struct SetsLds : UnionLds { CacheTile tile[2]; };

// What a lane holds of the 64 blocks of a list: the block, its members among the wave's tokens, and the factors
struct BlockLane {
    int block, members;
    float ck;        // c ks
    float lv, iv;    // log2(vs / w) and w / vs; SAFE: vs and 1
};

struct AttnState {
    f32x16 o[2];      // O^T [dim tile]
    float m, l;       // reference, and this lane's part of the sum
};

__device__ __forceinline__ int seq_tokens(const CacheAttnParams& p, int b) { return seq_keys(p, b); }

// x a + b in two roundings
__device__ __forceinline__ float times_plus(float x, float a, float b) {
#pragma clang fp contract(off)
    const float y = x * a;
    return y + b;
}

template <bool SAFE>
__device__ __forceinline__ void attend_tile(const CacheTile& t, const bf16x8 (&qf)[4], bool member, int valid, float ck, float lv, float iv,
                                            AttnState& a) {
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    auto keys = [&](int kt, int ds) { return as_bf16x8(ld16(t.K + ((kt * 4 + ds) * 64 + lane) * 8)); };
    auto vals = [&](int kt, int dt, int s2) { return as_bf16x8(ld16(t.V + (((kt * 2 + dt) * 2 + s2) * 64 + lane) * 8)); };
    f32x16 s[2] = {splat(0.f), splat(0.f)};
#pragma unroll
    for (int ds = 0; ds < 4; ++ds)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = mfma32(keys(kt, ds), qf[ds], s[kt]);
    if (valid < 64) {
        seldom();
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            int left = valid - 32 * kt - 16 * hh;
            asm volatile("" : "+v"(left));
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kt][e] = e < left ? s[kt][e] : -INFINITY;
        }
    }
    float mt = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mt = __builtin_elementwise_maximum(mt, s[kt][e]);
    const float shift = SAFE ? 0.f : lv;
    mt = fmaf(xor32_max(mt), ck, shift);
    const bool move = member && mt > a.m + kTau;
    if (__builtin_amdgcn_ballot_w64(move)) {
        const float alpha = move ? __builtin_amdgcn_exp2f(a.m - mt) : 1.f;
        a.m = move ? mt : a.m;
        a.o[0] *= alpha;
        a.o[1] *= alpha;
        a.l *= alpha;
    }
    const float ref = member ? shift - a.m : -INFINITY;   // P = 0 for the others
    // (of scores past 2^30 the fused form leaves more than fp32's exponents beside their rounded maximum)
    auto weight = [&](float x) { return __builtin_amdgcn_exp2f(SAFE ? times_plus(x, ck, ref) : fmaf(x, ck, ref)); };
    bf16x8 pb[2][2];
    float lt[2] = {0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = pack_bf16x2(weight(s[kt][8 * s2 + 2 * i]), weight(s[kt][8 * s2 + 2 * i + 1]));
            }
            pb[kt][s2] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
            lt[kt] = operand_sum(pb[kt][s2], lt[kt]);
        }
    if constexpr (SAFE) {
        if (member) a.l += lt[0] + lt[1];
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            f32x16 y = splat(0.f);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) y = mfma32(vals(kt, dt, s2), pb[kt][s2], y);
#pragma unroll
            for (int e = 0; e < 16; ++e) a.o[dt][e] = member ? fmaf(y[e], lv, a.o[dt][e]) : a.o[dt][e];
        }
    } else {
        a.l = fmaf(lt[0] + lt[1], iv, a.l);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) a.o[dt] = mfma32(vals(kt, dt, s2), pb[kt][s2], a.o[dt]);
    }
}

// Factors of a block's scales.  A scale of 0 stands for zeros only: any positive one does.
__device__ __forceinline__ float score_factor(float c, float ks) {
    return ks == 0.f ? 1.f : fminf(fmaxf(c * ks, FLT_MIN), FLT_MAX) + (ks - ks);   // (NaN stays)
}

__device__ __forceinline__ float wave_max_f(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

// Scales of values further than 2^60 from w are for the SAFE form.
constexpr float kSpread = 0x1p60f;

template <bool FP8, bool SAFE, typename Lds>
struct Walk {
    const CacheAttnParams& p;
    Lds& L;
    int b, h, end, sub;
    const bf16x8 (&qf)[4];
    const Row& row;
    AttnState& a;
    float w;        // 0: not chosen yet
    bool narrow;    // all scales of values within kSpread of w so far

    __device__ __forceinline__ void load(int block, int st, uint4& k, uint4& v) const {
        const int64_t from = block_at(p.cache, b, block, h) * (p.bs * 64) + st * kCodeTile + 16 * threadIdx.x;
        k = ld16(static_cast<const uint8_t*>(p.cache.k_codes) + from);
        v = ld16(static_cast<const uint8_t*>(p.cache.v_codes) + from);
    }
    __device__ __forceinline__ static void expand(bf16_t* at, const uint4& u) {   // 16 codes: two operands of a lane
        const uint2 a = codes_bf16<FP8>(u.x), b = codes_bf16<FP8>(u.y), c = codes_bf16<FP8>(u.z), d = codes_bf16<FP8>(u.w);
        *reinterpret_cast<uint4*>(at) = make_uint4(a.x, a.y, b.x, b.y);
        *reinterpret_cast<uint4*>(at + 64 * 8) = make_uint4(c.x, c.y, d.x, d.y);
    }
    __device__ __forceinline__ void put(int buf, const uint4& k, const uint4& v) const {
        const int tid = threadIdx.x, at = ((tid >> 6) * 2 * 64 + (tid & 63)) * 8;
        expand(L.tile[buf].K + at, k);
        expand(L.tile[buf].V + at, v);
    }
    // up to 64 blocks, lane i < count holding the i-th
    __device__ __forceinline__ void blocks(int count, int block, int members) {
        const int lane = threadIdx.x & 63;
        const int64_t at = block_at(p.cache, b, block, h);
        const float vs = p.cache.v_scale[at], ck = score_factor(p.c, p.cache.k_scale[at]);
        float lv, iv;
        if constexpr (SAFE) {
            lv = vs;
            iv = 1.f;
        } else {
            if (w == 0.f) {
                w = wave_max_f(vs > 0.f && vs < INFINITY ? vs : 0.f);
                if (w == 0.f) w = 1.f;
            }
            const float of = vs == 0.f ? w : vs;
            narrow = narrow && !__builtin_amdgcn_ballot_w64(!(of <= w * kSpread && of >= w * (1.f / kSpread)));
            iv = w / of;
            lv = __builtin_amdgcn_logf(of / w);
        }
        auto key0 = [&](int i) { return __builtin_amdgcn_readlane(block, i) * p.bs; };
        auto next = [&](int& i, int& st) {   // the tile after (i, st); i = count: none
            if (st + 1 < sub && key0(i) + 64 * (st + 1) < end) ++st;
            else {
                ++i;
                st = 0;
            }
        };
        uint4 kr, vr;
        int i = 0, st = 0, ni = 0, nst = 0;
        load(__builtin_amdgcn_readlane(block, 0), 0, kr, vr);
        put(0, kr, vr);
        next(ni, nst);
        if (ni < count) load(__builtin_amdgcn_readlane(block, ni), nst, kr, vr);
        for (int buf = 0; i < count; buf ^= 1) {
            lds_barrier();
            int fi = ni, fst = nst;
            if (ni < count) {
                put(buf ^ 1, kr, vr);
                next(fi, fst);
                if (fi < count) load(__builtin_amdgcn_readlane(block, fi), fst, kr, vr);
            }
            const uint32_t of = (uint32_t)__builtin_amdgcn_readlane(members, i);
            auto lane_f = [&](float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), i)); };
            if (of != 0)
                attend_tile<SAFE>(L.tile[buf], qf, row.in(of), min(64, end - key0(i) - 64 * st), lane_f(ck), lane_f(lv), lane_f(iv), a);
            i = ni; st = nst;
            ni = fi; nst = fst;
        }
        lds_barrier();   // the buffers are free for the next blocks
    }
};

template <bool FP8, bool DENSE, bool SAFE>
__device__ __forceinline__ bool attend(const CacheAttnParams& p, std::conditional_t<DENSE, DenseLds, SetsLds>& L, int b, int h, int n0, int split,
                                       const Row& row, const bf16x8 (&qf)[4], AttnState& a, float& w) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    a.o[0] = a.o[1] = splat(0.f);
    a.m = -FLT_MAX;   // finite, so that keys whose score is -inf are exp2(-inf) = 0 also before any other
    a.l = 0.f;
    const int end = seq_tokens(p, b);
    Walk<FP8, SAFE, std::remove_reference_t<decltype(L)>> walk{p, L, b, h, end, p.bs / 64, qf, row, a, 0.f, true};
    const int live = (int)(((int64_t)end + p.bs - 1) / p.bs);   // blocks with a key
    if constexpr (DENSE) {
        const int first = (int)((int64_t)live * split / p.splits), past = (int)((int64_t)live * (split + 1) / p.splits);
        for (int e0 = first; e0 < past; e0 += 64) walk.blocks(min(64, past - e0), min(e0 + lane, past - 1), -1);
    } else {
        const bool by_block = p.keys != nullptr;
        for (int c0 = 0; c0 < live; c0 += kUnion) {
            const int found = unite(p, L, b, h, n0, end, c0, min(kUnion, live - c0), split, by_block ? p.splits : 1);
            const int first = by_block ? 0 : (int)((uint32_t)(found * split) / (uint32_t)p.splits);
            const int past = by_block ? found : (int)((uint32_t)(found * (split + 1)) / (uint32_t)p.splits);
            for (int e0 = first; e0 < past; e0 += 64) {
                const int count = min(64, past - e0), u = L.list[e0 + min(lane, count - 1)];
                walk.blocks(count, c0 + u, (int)L.members[u][wave]);
            }
            __syncthreads();
        }
    }
    w = SAFE || walk.w == 0.f ? 1.f : walk.w;
    return walk.narrow;
}

template <bool FP8, bool DENSE>
__global__ __launch_bounds__(kThreads, 3) void cache_attn_kernel(CacheAttnParams p, int total) {
    __shared__ std::conditional_t<DENSE, DenseLds, SetsLds> L;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_runs(blockIdx.x, total);
    const int split = id % p.splits, tile_id = id / p.splits % p.qtiles, rest = id / p.splits / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * kWaves * p.QW;
    Row row;
    if constexpr (DENSE) row.init(p, [&](int i) { return min(n0 + i, p.Nq - 1); }, b, h, n0, wave, lane & 31);
    else {
        load_tokens(p, L, b, h, n0);
        row.init(p, [&](int i) { return L.tokens[i]; }, b, h, n0, wave, lane & 31);
    }
    bf16x8 qf[4];   // step ds: dims 32 (ds / 2) + 16 hh + 8 (ds % 2) .. (see qcache.h)
    const bf16_t* qr = p.q + b * p.q_sb + row.n * p.q_sn + row.head * p.q_sh + 16 * hh;
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) qf[ds] = as_bf16x8(ld16(qr + 32 * (ds >> 1) + 8 * (ds & 1)));
    arrived(qf);
    AttnState a;
    float w;
    bool ok = attend<FP8, DENSE, false>(p, L, b, h, n0, split, row, qf, a, w);
    ok = ok && finite(a.o[0]) && finite(a.o[1]) && a.l - a.l == 0.f;
    if (__syncthreads_or(!ok)) attend<FP8, DENSE, true>(p, L, b, h, n0, split, row, qf, a, w);
    const float l = xor32_add(a.l), f = l == 0.f ? 0.f : 1.f / l;
    if (!row.live) return;
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.B * p.Nq * p.Hq;
        float* d = p.part_o + (split * rows + row.at) * 64 + 4 * hh;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<float4*>(d + 32 * dt + 8 * g4) = make_float4(a.o[dt][4 * g4] * f * w, a.o[dt][4 * g4 + 1] * f * w,
                                                                               a.o[dt][4 * g4 + 2] * f * w, a.o[dt][4 * g4 + 3] * f * w);
        if (hh == 0) {
            int e = 0;
            const float part = frexpf(l, &e);   // (NaN and infinity stay what they are)
            p.part_ml[split * rows + row.at] = make_float2(a.m + (float)e, part);
        }
        return;
    }
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) a.o[dt] *= f;   // (before w: 1 / l and w / l need not fit together)
    store_row(p.out, row.at, lane, a.o, w);
}

// ------------------------------------------------------------------ few rows

// One token above all: no more than 16 rows (token, head) of a kv head.  A workgroup's waves take the tiles
// of 64 keys of its share in turn, straight from memory into the operands of v_mfma_f32_16x16x32_bf16
// (lane group g = lane / 16): in step m the keys' rows 4 g + i are tokens 16 g + 4 m + i, so that a lane
// ends with the scores of the 16 tokens that its chunk of the values holds.  A tile is requested while
// the one before is computed.
constexpr int kFewRows = 16, kFewEntries = 64;

struct FewState {
    f32x4 o[4];       // O^T [16 dims]: dims 16 dg + 4 g + i
    float m, l;
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
__device__ __forceinline__ void attend_few(const Codes& t, const bf16x8 (&qf)[2], bool member, int valid, float c, float& w, bool& narrow, FewState& a) {
    const int g = (threadIdx.x & 63) >> 4;
    const float ck = score_factor(c, t.ks);
    float lv = t.vs, iv = 1.f;
    if constexpr (!SAFE) {
        if (w == 0.f && t.vs > 0.f && t.vs < INFINITY) w = t.vs;
        const float base = w == 0.f ? 1.f : w, of = t.vs == 0.f ? base : t.vs;
        narrow = narrow && of <= base * kSpread && of >= base * (1.f / kSpread);
        iv = base / of;
        lv = __builtin_amdgcn_logf(of / base);
    }
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
    const float shift = SAFE ? 0.f : lv;
    mt = fmaf(xor32_max(xor16_max(mt)), ck, shift);
    const bool move = member && mt > a.m + kTau;
    if (__builtin_amdgcn_ballot_w64(move)) {
        const float alpha = move ? __builtin_amdgcn_exp2f(a.m - mt) : 1.f;
        a.m = move ? mt : a.m;
#pragma unroll
        for (int dg = 0; dg < 4; ++dg) a.o[dg] *= alpha;
        a.l *= alpha;
    }
    const float ref = member ? shift - a.m : -INFINITY;   // P = 0 for the others
    auto weight = [&](float x) { return __builtin_amdgcn_exp2f(SAFE ? times_plus(x, ck, ref) : fmaf(x, ck, ref)); };
    bf16x8 pb[2];
    float lt = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = pack_bf16x2(weight(s[2 * j + (i >> 1)][2 * (i & 1)]), weight(s[2 * j + (i >> 1)][2 * (i & 1) + 1]));
        pb[j] = as_bf16x8(make_uint4(u[0], u[1], u[2], u[3]));
        lt = operand_sum(pb[j], lt);
    }
    if constexpr (SAFE) {
        if (member) a.l += lt;
    } else a.l = fmaf(lt, iv, a.l);
#pragma unroll
    for (int dg = 0; dg < 4; ++dg) {
        const bf16x8 v0 = codes8<FP8>(t.v[dg].x, t.v[dg].y), v1 = codes8<FP8>(t.v[dg].z, t.v[dg].w);
        if constexpr (SAFE) {
            const f32x4 y = mfma16(v1, pb[1], mfma16(v0, pb[0], f32x4{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
            for (int i = 0; i < 4; ++i) a.o[dg][i] = member ? fmaf(y[i], lv, a.o[dg][i]) : a.o[dg][i];
        } else a.o[dg] = mfma16(v1, pb[1], mfma16(v0, pb[0], a.o[dg]));
    }
}

template <bool FP8, bool DENSE>
__global__ __launch_bounds__(kThreads, 3) void cache_attn_few_kernel(CacheAttnParams p) {
    __shared__ __attribute__((aligned(16))) float O[kWaves][kFewRows][64];
    __shared__ float2 ml[kWaves][kFewRows];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits, h = rest % p.Hk, b = rest / p.Hk;
    const int end = seq_keys(p, b), sub = p.bs / 64, rows = p.Nq * p.G;
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
    const int first = (int)((int64_t)units * split / p.splits), past = (int)((int64_t)units * (split + 1) / p.splits);
    const int kt = r >> 3, ko = kt * 2048 + (g >> 1) * 1024 + (g & 1) * 512 + (r & 7) * 16;
    const int vo = (g >> 1) * 2048 + (g & 1) * 512 + r * 16;
    // unit u: its first key, and the tokens that have it
    auto where = [&](int u, uint32_t& of) {
        of = ~0u;
        if constexpr (DENSE) return u * 64;
        else {
            const int which = (int)((uint32_t)u / (uint32_t)sub);
            const int src = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(lead && rank == which));
            of = (uint32_t)__builtin_amdgcn_readlane((int)tokens, src);
            return __builtin_amdgcn_readlane(blk, src) * p.bs + (u - which * sub) * 64;
        }
    };
    auto load = [&](int key0, Codes& t) {
        const int j = (int)((uint32_t)key0 / (uint32_t)p.bs);
        const int64_t at = block_at(p.cache, b, j, h), from = at * (p.bs * 64) + (key0 - j * p.bs) * 64;
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
    float w;
    bool narrow;
    auto walk = [&](auto safe) {
        w = 0.f;
        narrow = true;
#pragma unroll
        for (int dg = 0; dg < 4; ++dg) a.o[dg] = f32x4{0.f, 0.f, 0.f, 0.f};
        a.m = -FLT_MAX;
        a.l = 0.f;
        if (first + wave >= past) return;
        Codes next;
        uint32_t of_next;
        int key_next = where(first + wave, of_next);
        load(min(key_next, end - 1), next);   // (a block's later tiles may lie behind the end)
        for (int u = first + wave; u < past; u += kWaves) {
            const Codes t = next;
            const uint32_t of = of_next;
            const int key0 = key_next;
            if (u + kWaves < past) {
                key_next = where(u + kWaves, of_next);
                load(min(key_next, end - 1), next);
            }
            if (key0 < end)
                attend_few<FP8, decltype(safe)::value>(t, qf, row_live && (DENSE || (of >> token & 1)), min(64, end - key0), p.c, w, narrow, a);
        }
        if (decltype(safe)::value || w == 0.f) w = 1.f;
    };
    walk(std::false_type{});
    bool ok = narrow && a.l - a.l == 0.f;
#pragma unroll
    for (int dg = 0; dg < 4; ++dg)
#pragma unroll
        for (int i = 0; i < 4; ++i) ok = ok && a.o[dg][i] - a.o[dg][i] == 0.f;
    if (__builtin_amdgcn_ballot_w64(!ok)) walk(std::true_type{});   // (a wave by itself)
    const float l = xor32_add(xor16_add(a.l)), f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int dg = 0; dg < 4; ++dg)
        *reinterpret_cast<float4*>(&O[wave][r][(16 * dg + 4 * g) ^ (4 * r)]) =
            make_float4(a.o[dg][0] * f * w, a.o[dg][1] * f * w, a.o[dg][2] * f * w, a.o[dg][3] * f * w);
    if (g == 0) {
        int e = 0;
        const float part = frexpf(l, &e);
        ml[wave][r] = make_float2(a.m + (float)e, part);
    }
    __syncthreads();
    // 16 threads a row
    const int row = tid / 16, d = 4 * (tid % 16);
    if (row >= rows) return;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = ml[i][row].y == 0.f ? m : fmaxf(m, ml[i][row].x);
    float sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const float2 part = ml[i][row];
        const float4 x = *reinterpret_cast<const float4*>(&O[i][row][d ^ (4 * row)]);
        const float y = part.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(part.x - m) * part.y;   // 0: no key
        sum += y;
        o.x = fmaf(y, x.x, o.x); o.y = fmaf(y, x.y, o.y); o.z = fmaf(y, x.z, o.z); o.w = fmaf(y, x.w, o.w);
    }
    const float y = sum == 0.f ? 0.f : 1.f / sum;
    const int t = row / p.G;
    const int64_t at = ((int64_t)b * p.Nq + t) * p.Hq + h * p.G + row - t * p.G;
    if (p.splits == 1) {
        *reinterpret_cast<uint2*>(p.out + at * 64 + d) = make_uint2(pack_bf16x2(o.x * y, o.y * y), pack_bf16x2(o.z * y, o.w * y));
        return;
    }
    const int64_t all = (int64_t)p.B * p.Nq * p.Hq;
    *reinterpret_cast<float4*>(p.part_o + (split * all + at) * 64 + d) = make_float4(o.x * y, o.y * y, o.z * y, o.w * y);
    if (d == 0) {
        int e = 0;
        const float part = frexpf(sum, &e);
        p.part_ml[split * all + at] = make_float2(m + (float)e, part);
    }
}

// ------------------------------------------------------------------ joins

// Joins the splits' partials: 16 lanes a row, 4 dims each, and TEAM such groups a row that take its splits
// in turn (of few splits one, of many all 16 of a workgroup).
template <int TEAM>
__global__ __launch_bounds__(kThreads) void cache_attn_join_kernel(CacheAttnParams p, int64_t rows) {
    __shared__ __attribute__((aligned(16))) float4 part[16][16];
    __shared__ float ml[16], sums[16];
    const int group = threadIdx.x / 16, j = threadIdx.x % 16, d = 4 * j, of = group % TEAM;
    const int64_t at = (int64_t)blockIdx.x * (16 / TEAM) + group / TEAM, row = at < rows ? at : rows - 1;
    float m = -INFINITY;
    for (int s = of + TEAM * j; s < p.splits; s += 16 * TEAM) {
        const float2 x = p.part_ml[s * rows + row];
        m = x.y == 0.f ? m : fmaxf(m, x.x);   // l = 0: no key in that share
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    if constexpr (TEAM > 1) {
        if (j == 0) ml[group] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TEAM; ++i) m = fmaxf(m, ml[group / TEAM * TEAM + i]);
    }
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = of; s < p.splits; s += TEAM) {
        const float2 x = p.part_ml[s * rows + row];
        const float4 y = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * 64 + d);
        const float f = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - m) * x.y;
        l += f;
        o.x = fmaf(f, y.x, o.x); o.y = fmaf(f, y.y, o.y); o.z = fmaf(f, y.z, o.z); o.w = fmaf(f, y.w, o.w);
    }
    if constexpr (TEAM > 1) {
        part[group][j] = o;
        if (j == 0) sums[group] = l;
        __syncthreads();
        if (of != 0) return;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
#pragma unroll
        for (int i = 0; i < TEAM; ++i) {
            const float4 y = part[group + i][j];
            l += sums[group + i];
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
    }
    if (at >= rows) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + row * 64 + d) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
}

// ------------------------------------------------------------------ host

int check_call(const mosaic_kv_cache* cache, int32_t nq, int32_t hq, int32_t d, int32_t K) {
    if (int e = check_cache(cache)) return e;
    if (nq <= 0) return MOSAIC_ERR_SHAPE;
    if (d != kHeadDim) return MOSAIC_ERR_HEAD_DIM;
    if (hq <= 0 || hq % cache->num_kv_heads) return MOSAIC_ERR_HEADS;
    const int G = hq / cache->num_kv_heads;
    if (G > 16 || K > kMaxSelected) return MOSAIC_ERR_UNSUPPORTED;
    if (K < 0) return MOSAIC_ERR_BLOCK_COUNT;
    // ids of workgroups stay in 31 bits
    const int64_t per = kWaves * (kRows / G), tiles = ((int64_t)nq + per - 1) / per;
    if ((double)tiles * cache->num_kv_heads * cache->batch * kMaxSplit > 2147483647.0 || nq > 0x7fffffff - 1024) return MOSAIC_ERR_SHAPE;
    if (((double)nq / kKeyTokens + 1) * cache->num_kv_heads * cache->batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    return MOSAIC_OK;
}

constexpr int64_t kFewGroups = 1024, kFewTiles = 2;

int64_t groups_of(const mosaic_kv_cache& c, int32_t nq, int32_t hq) {
    const int64_t per = kWaves * (kRows / (hq / c.num_kv_heads));
    return (nq + per - 1) / per * c.num_kv_heads * c.batch;
}
// Whether the call is one of cache_attn_few_kernel
bool few(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    const int64_t rows = (int64_t)nq * (hq / c.num_kv_heads);
    return rows <= kFewRows && (int64_t)nq * K <= kFewEntries;
}
// Shares of the keys: below one workgroup per CU they are split.
int choose_split(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    const int64_t sub = c.block_size / 64;
    if (few(c, nq, hq, K)) {
        const int64_t wgs = (int64_t)c.num_kv_heads * c.batch, tiles = K > 0 ? nq * K * sub : c.num_blocks * sub;
        const int64_t s = kFewGroups / wgs, most = tiles / (kWaves * kFewTiles);
        const int64_t n = s < most ? s : most;
        return (int)(n < 1 ? 1 : n);
    }
    const int64_t wgs = groups_of(c, nq, hq), most = K > 0 ? (K < kMaxSplit ? K : kMaxSplit) : c.num_blocks;
    if (wgs >= 256) return 1;
    const int64_t s = (K > 0 ? 512 : 768) / wgs;
    return (int)(s < most ? s : most);
}
size_t part_bytes(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    const int s = choose_split(c, nq, hq, K);
    const size_t rows = s == 1 ? 0 : (size_t)c.batch * nq * hq;
    return up(s * rows * kHeadDim * sizeof(float)) + up(s * rows * sizeof(float2));
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

size_t mosaic_cache_attn_fwd_workspace_size(const mosaic_kv_cache* cache, int32_t num_queries, int32_t num_q_heads, int32_t block_count) {
    if (check_call(cache, num_queries, num_q_heads, kHeadDim, block_count) != MOSAIC_OK) return 0;
    return part_bytes(*cache, num_queries, num_q_heads, block_count) +
           (block_count > 0 && !few(*cache, num_queries, num_q_heads, block_count) ? order_bytes(cache->batch, num_queries, num_q_heads, cache->num_kv_heads) : 0);
}

int mosaic_cache_attn_fwd(mosaic_bnhd q, const mosaic_kv_cache* cache, const int64_t* block_indices, const int32_t* kv_lens,
                          int32_t num_queries, int32_t num_q_heads, int32_t head_dim, int32_t block_count, float softmax_scale,
                          void* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_call(cache, num_queries, num_q_heads, head_dim, block_count)) return e;
    if (!scale_ok(softmax_scale)) return MOSAIC_ERR_UNSUPPORTED;
    if (q.ptr == nullptr || out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if ((block_indices == nullptr) != (block_count == 0)) return MOSAIC_ERR_BLOCK_COUNT;
    if (!aligned(q.ptr, 16) || q.stride_b % 8 || q.stride_n % 8 || q.stride_h % 8) return MOSAIC_ERR_ALIGNMENT;
    if (!aligned(block_indices, 8) || !aligned(out, 16) || !aligned(kv_lens, 4)) return MOSAIC_ERR_ALIGNMENT;
    const size_t need = mosaic_cache_attn_fwd_workspace_size(cache, num_queries, num_q_heads, block_count);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256))) return MOSAIC_ERR_WORKSPACE;
    CacheAttnParams p{};
    p.cache = *cache;
    p.q = static_cast<const bf16_t*>(q.ptr); p.q_sb = q.stride_b; p.q_sn = q.stride_n; p.q_sh = q.stride_h;
    p.idx = block_indices; p.lens = kv_lens;
    p.B = cache->batch; p.Nq = num_queries; p.Nk = cache->capacity; p.Hq = num_q_heads; p.Hk = cache->num_kv_heads;
    p.G = p.Hq / p.Hk; p.QW = kRows / p.G; p.bs = cache->block_size; p.K = block_count; p.nb = cache->num_blocks;
    p.qtiles = (num_queries + kWaves * p.QW - 1) / (kWaves * p.QW);
    p.qw_inverse = (65536 + p.QW - 1) / p.QW;
    p.splits = choose_split(*cache, num_queries, num_q_heads, block_count);
    p.out = static_cast<bf16_t*>(out);
    p.c = (softmax_scale > 0.f ? softmax_scale : 0.125f) * kLog2e;
    int64_t rows = (int64_t)p.B * num_queries * num_q_heads;
    char* ws = static_cast<char*>(workspace);
    if (p.splits > 1) {
        p.part_o = reinterpret_cast<float*>(ws);
        p.part_ml = reinterpret_cast<float2*>(ws + up(p.splits * rows * kHeadDim * sizeof(float)));
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (block_count > 0 && !few(*cache, num_queries, num_q_heads, block_count)) {
        place_order(p, ws + part_bytes(*cache, num_queries, num_q_heads, block_count));
        if (int e = launch_order(p, s)) return e;
    }
    const bool fp8 = cache->code_type == MOSAIC_CODE_E4M3, small = few(*cache, num_queries, num_q_heads, block_count);
    int total = (small ? 1 : p.qtiles) * p.Hk * p.B * p.splits;
    void* args[] = {&p, &total};
    const void* fn = block_count > 0 ? (fp8 ? (const void*)&cache_attn_kernel<true, false> : (const void*)&cache_attn_kernel<false, false>)
                                     : (fp8 ? (const void*)&cache_attn_kernel<true, true> : (const void*)&cache_attn_kernel<false, true>);
    if (small)
        fn = block_count > 0 ? (fp8 ? (const void*)&cache_attn_few_kernel<true, false> : (const void*)&cache_attn_few_kernel<false, false>)
                             : (fp8 ? (const void*)&cache_attn_few_kernel<true, true> : (const void*)&cache_attn_few_kernel<false, true>);
    if (launch(fn, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (p.splits == 1) return MOSAIC_OK;
    void* jargs[] = {&p, &rows};
    const bool team = p.splits > 16;
    const void* join = team ? (const void*)&cache_attn_join_kernel<16> : (const void*)&cache_attn_join_kernel<1>;
    return launch(join, dim3((unsigned)(team ? rows : (rows + 15) / 16)), jargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
