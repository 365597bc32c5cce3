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

// Joins the splits' partials: 16 lanes a row, 4 dims each.  Lane j holds the weights of splits j and
// j + 16, so that no load waits for another.
__global__ __launch_bounds__(kThreads) void cache_attn_join_kernel(CacheAttnParams p, int64_t rows) {
    static_assert(kMaxSplit == 32, "two splits a lane");
    const int64_t at = (int64_t)blockIdx.x * 16 + threadIdx.x / 16, row = at < rows ? at : rows - 1;
    const int j = threadIdx.x % 16, d = 4 * j;
    float2 ml[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = j + 16 * i;
        ml[i] = s < p.splits ? p.part_ml[s * rows + row] : make_float2(-INFINITY, 0.f);
    }
    float m = fmaxf(ml[0].y == 0.f ? -INFINITY : ml[0].x, ml[1].y == 0.f ? -INFINITY : ml[1].x);
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    float a[2], l = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // l = 0: no key in that share
        a[i] = ml[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - m) * ml[i].y;
        l += a[i];
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l += __shfl_xor(l, x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int n = min(16, p.splits - 16 * i);
#pragma unroll 8
        for (int s = 0; s < n; ++s) {
            const float4 x = *reinterpret_cast<const float4*>(p.part_o + ((s + 16 * i) * rows + row) * 64 + d);
            const float f = __shfl(a[i], (threadIdx.x & 48) + s);
            o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
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

int64_t groups_of(const mosaic_kv_cache& c, int32_t nq, int32_t hq) {
    const int64_t per = kWaves * (kRows / (hq / c.num_kv_heads));
    return (nq + per - 1) / per * c.num_kv_heads * c.batch;
}
// Shares of the keys: below one workgroup per CU they are split, up to two per CU together.
int choose_split(const mosaic_kv_cache& c, int32_t nq, int32_t hq, int32_t K) {
    const int64_t wgs = groups_of(c, nq, hq), most = K > 0 ? K : c.num_blocks;
    if (wgs >= 256) return 1;
    int64_t s = 512 / wgs;
    if (s > kMaxSplit) s = kMaxSplit;
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
           (block_count > 0 ? order_bytes(cache->batch, num_queries, num_q_heads, cache->num_kv_heads) : 0);
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
    if (block_count > 0) {
        place_order(p, ws + part_bytes(*cache, num_queries, num_q_heads, block_count));
        if (int e = launch_order(p, s)) return e;
    }
    int total = p.qtiles * p.Hk * p.B * p.splits;
    void* args[] = {&p, &total};
    const bool fp8 = cache->code_type == MOSAIC_CODE_E4M3;
    const void* fn = block_count > 0 ? (fp8 ? (const void*)&cache_attn_kernel<true, false> : (const void*)&cache_attn_kernel<false, false>)
                                     : (fp8 ? (const void*)&cache_attn_kernel<true, true> : (const void*)&cache_attn_kernel<false, true>);
    if (launch(fn, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (p.splits == 1) return MOSAIC_OK;
    void* jargs[] = {&p, &rows};
    return launch((const void*)&cache_attn_join_kernel, dim3((unsigned)((rows + 15) / 16)), jargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
