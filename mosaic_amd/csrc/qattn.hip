// qattn.hip -- attention of query tokens over key blocks of their own, forward and backward (gfx950).
//
// Row (b, n, h) = query token n and kv head h, with K block indices (a set: an index counts once,
// one out of range not at all) and the G query heads of the group:
//   o = sum_u p_u v_u / l,  p_u = exp2(c q.k_u - m),  c = softmax_scale log2 e,  l = sum p_u
// over the keys u of the set's blocks, those past the sequence's length left out; a row without a
// key is zeros (lse -inf).  fp32 scores, maxima, sums and accumulators; P is rounded to bf16 for
// the PV product (an error of half a step of bf16 per term, as the output's own rounding).
//
// A workgroup takes 4 waves x QW = 16 / G neighbouring tokens of one kv head, a wave the 16 rows
// (token, head) of its tokens.  Its tokens' sets are united in LDS (one 16-bit token mask per wave
// and block), and the union's blocks are staged once, 64 keys at a time, for all four waves; a
// wave skips the blocks none of its tokens has.  Neighbouring tokens of a mesh mostly choose the
// same blocks, so the union is little longer than one set, and where they do not, a wave computes
// no more 16-row tiles than its tokens would one by one.
//
// Per tile of 64 keys, transposed so that a lane's 16 scores are one row's
// (v_mfma_f32_16x16x32_bf16):
//   S^T = K Q^T    A = K rows (16-byte LDS reads),  B = q (registers)
//   O^T = V^T P^T  A = V^T (transposing LDS reads), B = P, which S^T's accumulators already hold in
//                  operand order (contraction index (g, i) <-> keys 4 g + i, 16 + 4 g + i - 4)
// Rows that are no members of a block keep their state: the tile's product goes to accumulators of
// its own and is added under the row's predicate, so nothing a row did not choose -- infinities and
// NaN among it -- reaches it.
//
// Few queries: the union is split over workgroups and the partial (m, l, O) joined by a second
// kernel.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "bsa_common.h"
#include "lds_dma.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTileElems = 64 * 64;
constexpr int kUnion = 1024;       // blocks whose members are marked at a time
constexpr int kMaxSplit = 32;

typedef short v4i16 __attribute__((ext_vector_type(4)));

struct QueryAttnParams {
    const bf16_t* q; int64_t q_sb, q_sn, q_sh;
    const bf16_t* k; int64_t k_sb, k_sn, k_sh;
    const bf16_t* v; int64_t v_sb, v_sn, v_sh;
    const bf16_t* go; int64_t go_sb, go_sn, go_sh;   // gradient of the output (backward)
    const bf16_t* o;           // the forward's output, contiguous (backward)
    const int64_t* idx;        // [B, Nq, Hk, K]
    const int32_t* lens;       // [B] keys of each sequence, or null
    bf16_t* out;               // [B, Nq, Hq, 64]: the output, or grad q
    float* lse;                // [B, Nq, Hq], or null (forward: written, backward: read)
    float* part_o;             // [splits, rows, 64] (splits > 1)
    float2* part_ml;           // [splits, rows]
    float* nlse;               // backward: -lse / c and -sum(o do) of each row
    float* ndelta;
    uint32_t* marks;           // backward: [B, Hk, nb, words] bit n: token n has the block
    bf16_t* dk; bf16_t* dv;    // [B, Nk, Hk, 64]
    int B, Nq, Nk, Hq, Hk, G, QW, bs, K, nb, words;
    int qtiles, splits;
    float scale, c;
};

// 16-byte chunk c of row r of a 64-row tile lies at c ^ swz16(r).  Row reads take one chunk of 16
// consecutive rows at a time: over the rows of one parity (256 bytes of banks hold two rows) it is a
// permutation.  Transposing reads take two neighbouring chunks of 8 consecutive rows: over the four
// of one parity its upper bits differ.
__device__ __forceinline__ int swz16(int r) { return (((r >> 1) & 3) << 1) | ((r >> 3) & 1); }

__device__ __forceinline__ bf16x8 tr_pair(const bf16_t* lo, const bf16_t* hi) {
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) v4i16*)(lo)));
    const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) v4i16*)(hi)));
    return as_bf16x8(make_uint4(a.x, a.y, b.x, b.y));
}

__device__ __forceinline__ int seq_keys(const QueryAttnParams& p, int b) {
    return p.lens == nullptr ? p.Nk : min(max(p.lens[b], 0), p.Nk);
}

// LDS of the forward and grad-q kernels
struct RowsLds {
    __attribute__((aligned(1024))) bf16_t K[2][kTileElems];
    __attribute__((aligned(1024))) bf16_t V[2][kTileElems];
    uint32_t members[kUnion][2];   // wave w: 16 bits at 16 (w % 2) of word w / 2
    uint16_t list[kUnion];
    int found[kWaves];
};

// Marks the members of blocks [c0, c0 + nc) among the workgroup's tokens n0 .. and lists the
// blocks that have any, ascending; returns their number.  Ends with a barrier.
__device__ __forceinline__ int unite(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, int end, int c0, int nc) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < nc; i += kThreads) L.members[i][0] = L.members[i][1] = 0;
    __syncthreads();
    const int tokens = min(kWaves * p.QW, p.Nq - n0);
    for (int e = tid; e < tokens * p.K; e += kThreads) {
        const int t = e / p.K, kk = e - t * p.K;
        const int64_t blk = p.idx[(((int64_t)b * p.Nq + n0 + t) * p.Hk + h) * p.K + kk] - c0;
        if (blk >= 0 && blk < nc && (c0 + blk) * p.bs < end) {
            const int w = t / p.QW;
            atomicOr(&L.members[blk][w >> 1], 1u << (16 * (w & 1) + t - w * p.QW));
        }
    }
    __syncthreads();
    const int per = (nc + kThreads - 1) / kThreads * 64;   // blocks a wave lists
    int n = 0;
    for (int i = wave * per + lane; i - lane < (wave + 1) * per; i += 64)
        n += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < nc && (L.members[i][0] | L.members[i][1])));
    if (lane == 0) L.found[wave] = n;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        at += w < wave ? L.found[w] : 0;
        total += L.found[w];
    }
    for (int i = wave * per + lane; i - lane < (wave + 1) * per; i += 64) {
        const bool on = i < nc && (L.members[i][0] | L.members[i][1]);
        const uint64_t m = __builtin_amdgcn_ballot_w64(on);
        if (on) L.list[at + (int)__builtin_popcountll(m & ((1ull << lane) - 1ull))] = (uint16_t)i;
        at += (int)__builtin_popcountll(m);
    }
    __syncthreads();
    return total;
}

// Requests keys key0 .. key0 + 63 into one buffer; rows past the sequence's end repeat its last
// one.  Each wave loads 16 rows of K and V; addresses are 64-bit throughout.
__device__ __forceinline__ void stage(const QueryAttnParams& p, const bf16_t* kb, const bf16_t* vb, int key0, int end,
                                      bf16_t* Kd, bf16_t* Vd, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row0 = 16 * wave + 8 * i, row = row0 + (lane >> 3);
        const int64_t key = min(key0 + row, end - 1);
        const int chunk = 8 * ((lane & 7) ^ swz16(row));
        dma16_at(kb + key * p.k_sn + chunk, lds_addr(Kd + row0 * 64));
        dma16_at(vb + key * p.v_sn + chunk, lds_addr(Vd + row0 * 64));
    }
}

// Per-lane LDS element offsets of the operand reads
struct RowReads {
    int row[2];   // row c16, chunk 4 ks + g; + 16 kt * 64
    int tr[4];    // transposing read of dims 16 dt ..: row 4 g + s / 4, + (32 c + 16 half) * 64
    __device__ __forceinline__ void init(int lane) {
        const int s = lane & 15, g = lane >> 4, r = 4 * g + (s >> 2);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) row[ks] = s * 64 + 8 * ((4 * ks + g) ^ swz16(s));
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) tr[dt] = r * 64 + 8 * ((2 * dt + ((s & 3) >> 1)) ^ swz16(r)) + 4 * (s & 1);
    }
};

// acc^T[key tile] = T rows . B^T over 64 dims, from `start`
__device__ __forceinline__ void row_products(const bf16_t* T, const RowReads& rr, const bf16x8 (&b)[2], float start, f32x4 (&acc)[4]) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[kt][e] = start;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
            acc[kt] = mfma16(as_bf16x8(*reinterpret_cast<const uint4*>(T + 16 * kt * 64 + rr.row[ks])), b[ks], acc[kt]);
    }
}

// acc^T[dim tile] += T^T . B^T over 64 keys, B in the accumulator order of row_products
__device__ __forceinline__ void col_products(const bf16_t* T, const RowReads& rr, const bf16x8 (&b)[2], f32x4 (&acc)[4]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
            acc[dt] = mfma16(tr_pair(T + 32 * c * 64 + rr.tr[dt], T + (32 * c + 16) * 64 + rr.tr[dt]), b[c], acc[dt]);
}

__device__ __forceinline__ float row_add(float x) {   // over the four lanes of a row
    x += __shfl_xor(x, 16);
    return xor32_add(x);
}
__device__ __forceinline__ float row_max(float x) { return xor32_max(fmaxf(x, __shfl_xor(x, 16))); }

// The rows of a wave, one per column c16 = lane % 16: token and query head, and its place in [B, Nq, Hq]
struct Row {
    int token, head;   // token within the wave
    bool live;
    int64_t n, at;
    __device__ __forceinline__ void init(const QueryAttnParams& p, int b, int h, int wave_n0, int lane) {
        const int r = lane & 15;
        token = r / p.G;
        live = token < p.QW && wave_n0 + token < p.Nq;
        head = h * p.G + (live ? r - token * p.G : 0);
        n = live ? wave_n0 + token : min(wave_n0, p.Nq - 1);
        at = ((int64_t)b * p.Nq + n) * p.Hq + head;
    }
};

__device__ __forceinline__ void load_row(const bf16_t* x, int64_t sb, int64_t sn, int64_t sh, int b, const Row& r, int lane, bf16x8 (&f)[2]) {
    const bf16_t* at = x + b * sb + r.n * sn + r.head * sh + 8 * (lane >> 4);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) f[ks] = as_bf16x8(ld16(at + 32 * ks));
}

__device__ __forceinline__ void store_row(bf16_t* out, int64_t at, int lane, const f32x4 (&o)[4], float f) {
    bf16_t* d = out + at * 64 + 4 * (lane >> 4);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
        *reinterpret_cast<uint2*>(d + 16 * dt) =
            make_uint2(pack_bf16x2(o[dt][0] * f, o[dt][1] * f), pack_bf16x2(o[dt][2] * f, o[dt][3] * f));
}

// Runs `tile(K, V, members of this wave, valid keys)` over the tiles of this workgroup's share of
// the union, staged in two buffers with one barrier each.
template <typename Tile>
__device__ __forceinline__ void for_tiles(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, int split, int splits, Tile tile) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int end = seq_keys(p, b), sub = p.bs / 64;
    const bf16_t* kb = p.k + b * p.k_sb + h * p.k_sh;
    const bf16_t* vb = p.v + b * p.v_sb + h * p.v_sh;
    const int live = (int)min((int64_t)p.nb, ((int64_t)end + p.bs - 1) / p.bs);   // blocks with a key
    for (int c0 = 0; c0 < live; c0 += kUnion) {
        const int found = unite(p, L, b, h, n0, end, c0, min(kUnion, live - c0));
        const int first = (int)((int64_t)found * split / splits), past = (int)((int64_t)found * (split + 1) / splits);
        const int tiles = (past - first) * sub;
        auto key_of = [&](int t) { return (c0 + __builtin_amdgcn_readfirstlane((int)L.list[first + t / sub])) * p.bs + t % sub * 64; };
        // tiles past the end are only in the union's last block
        if (tiles > 0) stage(p, kb, vb, key_of(0), end, L.K[0], L.V[0], wave, lane);
        for (int t = 0; t < tiles; ++t) {
            const int key0 = key_of(t), valid = min(64, end - key0);
            wait_vmem();
            lds_barrier();
            if (t + 1 < tiles && key_of(t + 1) < end) stage(p, kb, vb, key_of(t + 1), end, L.K[(t + 1) & 1], L.V[(t + 1) & 1], wave, lane);
            if (valid <= 0) break;
            if (valid < 64) {   // zeros behind the last key: what P = 0 multiplies there
                for (int i = threadIdx.x; i < (64 - valid) * 8; i += kThreads)
                    *reinterpret_cast<uint4*>(L.V[t & 1] + (valid + i / 8) * 64 + i % 8 * 8) = make_uint4(0, 0, 0, 0);
                lds_barrier();
            }
            const int u = L.list[first + t / sub];
            const uint32_t mine = (L.members[u][wave >> 1] >> (16 * (wave & 1))) & 0xffffu;
            const uint32_t m = __builtin_amdgcn_readfirstlane(mine);
            if (m != 0) tile(L.K[t & 1], L.V[t & 1], m, valid);
        }
        wait_vmem();
        __syncthreads();   // the lists and buffers are free for the next blocks
    }
}

__global__ __launch_bounds__(kThreads) void query_attn_kernel(QueryAttnParams p, int total) {
    __shared__ RowsLds L;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_remap(blockIdx.x, total);
    const int split = id % p.splits, tile_id = id / p.splits % p.qtiles, rest = id / p.splits / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * kWaves * p.QW;
    Row row;
    row.init(p, b, h, n0 + wave * p.QW, lane);
    bf16x8 qf[2];
    load_row(p.q, p.q_sb, p.q_sn, p.q_sh, b, row, lane, qf);
    RowReads rr;
    rr.init(lane);
    f32x4 o[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for_tiles(p, L, b, h, n0, split, p.splits, [&](const bf16_t* Kt, const bf16_t* Vt, uint32_t members, int valid) {
        f32x4 s[4];
        row_products(Kt, rr, qf, 0.f, s);
        if (valid < 64) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[kt][e] = 16 * kt + 4 * g + e < valid ? s[kt][e] : -INFINITY;
        }
        float mt = s[0][0];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[kt][e]);
        const float mnew = fmaxf(m, row_max(mt) * p.c);
        bf16x8 pb[2];
        float lt = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4& x = s[2 * c + i / 2];
                const float p0 = __builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1)], p.c, -mnew));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1) + 1], p.c, -mnew));
                lt += p0 + p1;
                w[i] = pack_bf16x2(p0, p1);
            }
            pb[c] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
        }
        f32x4 add[4];
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) add[dt][e] = 0.f;
        col_products(Vt, rr, pb, add);
        if (row.live && (members >> row.token & 1)) {
            const float alpha = __builtin_amdgcn_exp2f(m - mnew);
            m = mnew;
            l = fmaf(l, alpha, lt);
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[dt][e] = fmaf(o[dt][e], alpha, add[dt][e]);
        }
    });
    l = row_add(l);
    if (!row.live) return;
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.B * p.Nq * p.Hq;
        float* d = p.part_o + (split * rows + row.at) * 64 + 4 * g;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) *reinterpret_cast<float4*>(d + 16 * dt) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
        if (g == 0) p.part_ml[split * rows + row.at] = make_float2(m, l);
        return;
    }
    // a row without a key has l = 0 (any other at least the largest score's 1, or NaN)
    store_row(p.out, row.at, lane, o, l == 0.f ? 0.f : 1.f / l);
    if (p.lse != nullptr && g == 0) p.lse[row.at] = m + __builtin_amdgcn_logf(l);
}

// Joins the splits' partials: 16 lanes a row, 4 dims each.
__global__ __launch_bounds__(kThreads) void query_attn_join_kernel(QueryAttnParams p, int64_t rows) {
    const int64_t row = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (row >= rows) return;
    const int d = threadIdx.x % 16 * 4;
    float m = -INFINITY;
    for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[s * rows + row].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
        const float2 ml = p.part_ml[s * rows + row];
        if (ml.y == 0.f) continue;          // no key in this share
        const float a = __builtin_amdgcn_exp2f(ml.x - m);
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * 64 + d);
        l = fmaf(a, ml.y, l);
        o.x = fmaf(a, x.x, o.x); o.y = fmaf(a, x.y, o.y); o.z = fmaf(a, x.z, o.z); o.w = fmaf(a, x.w, o.w);
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + row * 64 + d) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
    if (p.lse != nullptr && d == 0) p.lse[row] = m + __builtin_amdgcn_logf(l);
}

// ------------------------------------------------------------------ backward
// delta = sum_d o do;  P = exp2(c q.k - lse);  dS = P (do.v - delta)
//   dq = scale sum_u dS k_u,   dk_u = scale sum over the rows that have u of dS q,   dv_u = sum P do
// P and dS are rounded to bf16 for their products, everything else is fp32.

// grad q: the forward's loop.  Also writes -lse / c (what the scores accumulate onto, so that
// exp2(c s) is P) and -delta of every row for grad k / v.
//
// sum_u dS_u = 0, so what all the keys of a row share cancels in dq, and errors of dS that do not
// cancel multiply it: keys chosen together share much.  With B = sum P k and dS' the rounded dS,
//   dq = scale (sum dS' k - (sum dS') B)
// takes that part out: the first guess of delta comes from the rounded output and need not be exact
// here, and the exact one, delta + sum P (do.v - delta), goes to grad k / v.  One product more per
// tile on operands at hand; without it grad q at 12288 tokens of nside 32 (12 blocks of 64) is
// 5.1e-3 off (2-norm), with it 2.4e-3 (the output's own rounding alone: 1.7e-3).
__global__ __launch_bounds__(kThreads) void query_attn_dq_kernel(QueryAttnParams p, int total) {
    __shared__ RowsLds L;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_remap(blockIdx.x, total);
    const int tile_id = id % p.qtiles, rest = id / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * kWaves * p.QW;
    Row row;
    row.init(p, b, h, n0 + wave * p.QW, lane);
    bf16x8 qf[2], gf[2];
    load_row(p.q, p.q_sb, p.q_sn, p.q_sh, b, row, lane, qf);
    load_row(p.go, p.go_sb, p.go_sn, p.go_sh, b, row, lane, gf);
    float delta = 0.f;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const uint4 ov = ld16(p.o + row.at * 64 + 32 * ks + 8 * g), gv = __builtin_bit_cast(uint4, gf[ks]);
        const uint32_t ow[4] = {ov.x, ov.y, ov.z, ov.w}, gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) delta = fmaf(bf_lo(ow[i]), bf_lo(gw[i]), fmaf(bf_hi(ow[i]), bf_hi(gw[i]), delta));
    }
    delta = row_add(delta);
    const float nlse = -p.lse[row.at] / p.c;
    RowReads rr;
    rr.init(lane);
    const bf16x8 ones = as_bf16x8(make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
    f32x4 dq[4], kbar[4], sum = {0.f, 0.f, 0.f, 0.f};   // sum dS' k, sum P k, sum dS'
    float rest_d = 0.f;                                  // this lane's part of sum P (do.v - delta)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) dq[dt][e] = kbar[dt][e] = 0.f;
    for_tiles(p, L, b, h, n0, 0, 1, [&](const bf16_t* Kt, const bf16_t* Vt, uint32_t members, int valid) {
        f32x4 s[4], dp[4];
        row_products(Kt, rr, qf, nlse, s);
        row_products(Vt, rr, gf, -delta, dp);
        if (valid < 64) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool on = 16 * kt + 4 * g + e < valid;
                    s[kt][e] = on ? s[kt][e] : -INFINITY;
                    dp[kt][e] = on ? dp[kt][e] : 0.f;
                }
        }
        bf16x8 pb[2], db[2];
        float dsum = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t w[4], x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int kt = 2 * c + i / 2, e = 2 * (i & 1);
                const float p0 = __builtin_amdgcn_exp2f(s[kt][e] * p.c), p1 = __builtin_amdgcn_exp2f(s[kt][e + 1] * p.c);
                const float d0 = p0 * dp[kt][e], d1 = p1 * dp[kt][e + 1];
                dsum += d0 + d1;
                w[i] = pack_bf16x2(p0, p1);
                x[i] = pack_bf16x2(d0, d1);
            }
            pb[c] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
            db[c] = as_bf16x8(make_uint4(x[0], x[1], x[2], x[3]));
        }
        f32x4 dqt[4], kt_[4], st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) dqt[dt][e] = kt_[dt][e] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            st = mfma16(ones, db[c], st);
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const bf16x8 kT = tr_pair(Kt + 32 * c * 64 + rr.tr[dt], Kt + (32 * c + 16) * 64 + rr.tr[dt]);
                dqt[dt] = mfma16(kT, db[c], dqt[dt]);
                kt_[dt] = mfma16(kT, pb[c], kt_[dt]);
            }
        }
        if (row.live && (members >> row.token & 1)) {
            rest_d += dsum;
            sum += st;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                dq[dt] += dqt[dt];
                kbar[dt] += kt_[dt];
            }
        }
    });
    rest_d = row_add(rest_d);
    if (!row.live) return;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) dq[dt][e] = fmaf(-sum[0], kbar[dt][e], dq[dt][e]);
    store_row(p.out, row.at, lane, dq, p.scale);
    if (g == 0) {
        p.nlse[row.at] = nlse;
        p.ndelta[row.at] = -(delta + rest_d);
    }
}

// The tokens of each block, as bits: a workgroup takes 512 tokens (16 words) of one kv head and up
// to kUnion blocks, marks in LDS and writes every word, so nothing needs clearing and no order of
// atomics reaches memory.
constexpr int kMarkTokens = 512, kMarkWords = kMarkTokens / 32;
__global__ __launch_bounds__(kThreads) void query_marks_kernel(QueryAttnParams p, int groups) {
    __shared__ __attribute__((aligned(16))) uint32_t bits[kUnion * kMarkWords];
    const int grp = blockIdx.x % groups, rest = blockIdx.x / groups;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int c0 = blockIdx.y * kUnion, nc = min(kUnion, p.nb - c0);
    for (int i = threadIdx.x; i < nc * kMarkWords; i += kThreads) bits[i] = 0;
    __syncthreads();
    const int n0 = grp * kMarkTokens, tokens = min(kMarkTokens, p.Nq - n0);
    for (int e = threadIdx.x; e < tokens * p.K; e += kThreads) {
        const int t = e / p.K, kk = e - t * p.K;
        const int64_t blk = p.idx[(((int64_t)b * p.Nq + n0 + t) * p.Hk + h) * p.K + kk] - c0;
        if (blk >= 0 && blk < nc) atomicOr(&bits[blk * kMarkWords + t / 32], 1u << (t % 32));
    }
    __syncthreads();
    uint32_t* out = p.marks + (((int64_t)b * p.Hk + h) * p.nb + c0) * p.words + grp * kMarkWords;
    for (int i = threadIdx.x; i < nc * (kMarkWords / 4); i += kThreads) {
        const int blk = i / (kMarkWords / 4), w = i % (kMarkWords / 4) * 4;
        *reinterpret_cast<uint4*>(out + (int64_t)blk * p.words + w) = *reinterpret_cast<const uint4*>(bits + blk * kMarkWords + w);
    }
}

// grad k, grad v.  One workgroup = 64 keys of one kv head: it walks the tokens that have the block,
// QS = 64 / G at a time (64 rows of q and do gathered straight into LDS).  Wave w = (key half w / 2,
// row half w % 2) forms S = q k^T and dP = do v^T of its 32 rows x 32 keys
// (v_mfma_f32_32x32x16_bf16); P and dS stay in registers as the B operands of dV^T += do^T P and
// dK^T += q^T dS, whose A operands are transposing LDS reads.  The row halves are added at the end.
constexpr int kSegWords = 128;                 // words of marks listed at a time: 4096 tokens
constexpr int kListed = 32 * kSegWords + 64;   // and what was left of the last ones

__device__ __forceinline__ int swz32(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

struct KeysLds {
    __attribute__((aligned(1024))) bf16_t q[2][kTileElems];
    __attribute__((aligned(1024))) bf16_t g[2][kTileElems];
    float nlse[2][64], ndelta[2][64];
    int list[kListed];
    int sums[2];
};

__global__ __launch_bounds__(kThreads, 2) void query_attn_dkv_kernel(QueryAttnParams p, int tiles, int total) {
    __shared__ KeysLds L;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), kh = w >> 1, qh = w & 1;
    const int id = xcd_remap(blockIdx.x, total);
    const int kt = id % tiles, rest = id / tiles, h = rest % p.Hk, b = rest / p.Hk;
    const int key0 = kt * 64, end = seq_keys(p, b);
    const uint32_t* marks = p.marks + (((int64_t)b * p.Hk + h) * p.nb + key0 / p.bs) * p.words;
    const int QS = 64 / p.G;

    f32x16 dkT[2], dvT[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) { dkT[0][e] = 0.f; dkT[1][e] = 0.f; dvT[0][e] = 0.f; dvT[1][e] = 0.f; }
    int rd[4], tr[2][2];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) rd[kk] = r * 64 + 8 * ((2 * kk + hh) ^ swz32(r));
    {
        const int s4 = lane & 15, half = (lane >> 4) & 1;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int sec = 0; sec < 2; ++sec) {
                const int row = 4 * hh + (s4 >> 2) + 8 * sec;
                tr[dt][sec] = row * 64 + 8 * ((4 * dt + 2 * half + ((s4 & 3) >> 1)) ^ swz32(row)) + 4 * (s4 & 1);
            }
    }
    // rows of this lane's loads: 16 w + 8 i + lane / 8 (q, do), 16 w + lane (statistics)
    int ltok[3], lhead[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int row = i < 2 ? 16 * w + 8 * i + (lane >> 3) : 16 * w + (lane & 15);
        ltok[i] = min(row / p.G, QS - 1);
        lhead[i] = h * p.G + row % p.G;
    }
    if (key0 < end) {
        bf16x8 kf[4], vf[4];   // this wave's keys: row 32 kh + r (the last one again past the end), dims 16 kk + 8 hh ..
        {
            const int64_t key = min(key0 + 32 * kh + r, end - 1);
            const bf16_t* kr = p.k + b * p.k_sb + key * p.k_sn + h * p.k_sh + 8 * hh;
            const bf16_t* vr = p.v + b * p.v_sb + key * p.v_sn + h * p.v_sh + 8 * hh;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                kf[kk] = as_bf16x8(ld16(kr + 16 * kk));
                vf[kk] = as_bf16x8(ld16(vr + 16 * kk));
            }
        }
        const bf16_t* qb = p.q + b * p.q_sb;
        const bf16_t* gb = p.go + b * p.go_sb;
        // step s's rows into buffer s & 1; entries past the list repeat its last one
        auto request = [&](int s, int count) {
            const int buf = s & 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t n = L.list[min(s * QS + ltok[i], count - 1)];
                const int row0 = 16 * w + 8 * i, row = row0 + (lane >> 3);
                const int chunk = 8 * ((lane & 7) ^ swz32(row));
                dma16_at(qb + n * p.q_sn + lhead[i] * p.q_sh + chunk, lds_addr(L.q[buf] + row0 * 64));
                dma16_at(gb + n * p.go_sn + lhead[i] * p.go_sh + chunk, lds_addr(L.g[buf] + row0 * 64));
            }
            const int64_t at = ((int64_t)b * p.Nq + L.list[min(s * QS + ltok[2], count - 1)]) * p.Hq + lhead[2];
            if (lane < 16) {
                dma4_at(p.nlse + at, lds_addr(L.nlse[buf] + 16 * w));
                dma4_at(p.ndelta + at, lds_addr(L.ndelta[buf] + 16 * w));
            }
        };
        auto tr_read = [&](const bf16_t* T, int q0, int dt) { return tr_pair(T + q0 * 64 + tr[dt][0], T + q0 * 64 + tr[dt][1]); };
        auto step = [&](int buf, int rows) {
            const bf16_t* Qc = L.q[buf];
            const bf16_t* Gc = L.g[buf];
            f32x16 s, dp;
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const float4 l4 = *reinterpret_cast<const float4*>(L.nlse[buf] + 32 * qh + 8 * g4 + 4 * hh);
                const float4 d4 = *reinterpret_cast<const float4*>(L.ndelta[buf] + 32 * qh + 8 * g4 + 4 * hh);
                s[4 * g4] = l4.x; s[4 * g4 + 1] = l4.y; s[4 * g4 + 2] = l4.z; s[4 * g4 + 3] = l4.w;
                dp[4 * g4] = d4.x; dp[4 * g4 + 1] = d4.y; dp[4 * g4 + 2] = d4.z; dp[4 * g4 + 3] = d4.w;
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                s = mfma32(as_bf16x8(*reinterpret_cast<const uint4*>(Qc + 32 * qh * 64 + rd[kk])), kf[kk], s);
                dp = mfma32(as_bf16x8(*reinterpret_cast<const uint4*>(Gc + 32 * qh * 64 + rd[kk])), vf[kk], dp);
            }
            bf16x8 pb[2], db[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float pr = __builtin_amdgcn_exp2f(s[e] * p.c), ds = pr * dp[e];
                if (rows < 64) {   // rows past the list, or past QS G
                    const bool on = 32 * qh + 8 * (e >> 2) + 4 * hh + (e & 3) < rows;
                    pr = on ? pr : 0.f;
                    ds = on ? ds : 0.f;
                }
                pb[e >> 3][e & 7] = (__bf16)pr;
                db[e >> 3][e & 7] = (__bf16)ds;
            }
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) {
                    dvT[dt] = mfma32(tr_read(Gc, 32 * qh + 16 * ch, dt), pb[ch], dvT[dt]);
                    dkT[dt] = mfma32(tr_read(Qc, 32 * qh + 16 * ch, dt), db[ch], dkT[dt]);
                }
        };
        int count = 0;   // tokens listed
        for (int w0 = 0; w0 < p.words; w0 += kSegWords) {
            // list the tokens of words w0 .. behind the ones left over: waves 0 and 1, a word per lane
            const uint32_t word = w < 2 && w0 + tid < p.words ? marks[w0 + tid] : 0;
            int before = __builtin_popcount(word);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int x = __shfl_up(before, d);
                before += lane >= d ? x : 0;
            }
            if (w < 2 && lane == 63) L.sums[w] = before;
            __syncthreads();
            if (w < 2) {
                int at = count + before - __builtin_popcount(word) + (w == 1 ? L.sums[0] : 0);
                for (uint32_t m = word; m != 0; m &= m - 1) L.list[at++] = 32 * (w0 + tid) + __builtin_ctz(m);
            }
            count += L.sums[0] + L.sums[1];
            __syncthreads();
            const bool last = w0 + kSegWords >= p.words;
            const int steps = last ? (count + QS - 1) / QS : count / QS;
            if (steps > 0) request(0, count);
            for (int s = 0; s < steps; ++s) {
                wait_vmem();
                lds_barrier();
                if (s + 1 < steps) request(s + 1, count);
                step(s & 1, min(QS, count - s * QS) * p.G);
            }
            // the tokens left over go to the list's front
            const int rest_n = count - steps * QS;
            int keep = 0;
            if (tid < rest_n) keep = L.list[steps * QS + tid];
            __syncthreads();
            if (tid < rest_n) L.list[tid] = keep;
            count = rest_n > 0 ? rest_n : 0;
        }
        __syncthreads();
        // the row halves' sums: qh = 1 parks its accumulators in the buffers
        float* red = reinterpret_cast<float*>((kh == 0 ? L.q[0] : L.g[0]) + hh * kTileElems) + r;
        if (qh == 1) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                red[32 * e] = dkT[0][e];
                red[32 * (16 + e)] = dkT[1][e];
                red[32 * (32 + e)] = dvT[0][e];
                red[32 * (48 + e)] = dvT[1][e];
            }
        }
        __syncthreads();
        if (qh == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dkT[0][e] += red[32 * e];
                dkT[1][e] += red[32 * (16 + e)];
                dvT[0][e] += red[32 * (32 + e)];
                dvT[1][e] += red[32 * (48 + e)];
            }
        }
    }
    const int key = key0 + 32 * kh + r;
    if (qh == 0 && key < p.Nk) {   // zeros for keys past the sequence's end
        const int64_t base = (((int64_t)b * p.Nk + key) * p.Hk + h) * 64;
        const bool on = key < end;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                float kx[4], vx[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    kx[i] = on ? dkT[dt][4 * g4 + i] * p.scale : 0.f;
                    vx[i] = on ? dvT[dt][4 * g4 + i] : 0.f;
                }
                const int d = 32 * dt + 8 * g4 + 4 * hh;
                *reinterpret_cast<uint2*>(p.dk + base + d) = make_uint2(pack_bf16x2(kx[0], kx[1]), pack_bf16x2(kx[2], kx[3]));
                *reinterpret_cast<uint2*>(p.dv + base + d) = make_uint2(pack_bf16x2(vx[0], vx[1]), pack_bf16x2(vx[2], vx[3]));
            }
    }
}

// ------------------------------------------------------------------ host

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

int check_rows(const mosaic_bnhd& t) {
    if (t.ptr == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!aligned(t.ptr, 16) || t.stride_b % 8 || t.stride_n % 8 || t.stride_h % 8) return MOSAIC_ERR_ALIGNMENT;
    return MOSAIC_OK;
}

int check_shape(int32_t batch, int32_t nq, int32_t nk, int32_t hq, int32_t hk, int32_t d, int32_t bs, int32_t K) {
    if (batch <= 0 || nq <= 0 || nk <= 0) return MOSAIC_ERR_SHAPE;
    if (d != kHeadDim) return MOSAIC_ERR_HEAD_DIM;
    if (hq <= 0 || hk <= 0 || hq % hk) return MOSAIC_ERR_HEADS;
    if (hq / hk > 16) return MOSAIC_ERR_UNSUPPORTED;
    if (bs <= 0 || bs % 64) return MOSAIC_ERR_BLOCK_SIZE;
    if (K <= 0) return MOSAIC_ERR_BLOCK_COUNT;
    if (K > kMaxSelected) return MOSAIC_ERR_UNSUPPORTED;
    // ids of workgroups and keys stay in 31 bits
    if (nk > 0x7fffffff - bs || nq > 0x7fffffff - kMarkTokens) return MOSAIC_ERR_SHAPE;
    const int64_t qw = 16 / (hq / hk), tiles = ((int64_t)nq + 4 * qw - 1) / (4 * qw);
    if ((double)tiles * hk * batch * kMaxSplit > 2147483647.0) return MOSAIC_ERR_SHAPE;
    if ((double)((nk + 63) / 64) * hk * batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    return MOSAIC_OK;
}

// Workgroups of one share: below one per CU the union is split, up to two per CU together.
int choose_split(int32_t batch, int32_t nq, int32_t hq, int32_t hk, int32_t K) {
    const int64_t per = 4 * (16 / (hq / hk));
    const int64_t wgs = (nq + per - 1) / per * hk * batch;
    if (wgs >= 256) return 1;
    const int64_t s = 512 / wgs;
    return (int)(s < K ? (s < kMaxSplit ? s : kMaxSplit) : (K < kMaxSplit ? K : kMaxSplit));
}

void fill(QueryAttnParams& p, const mosaic_bnhd& q, const mosaic_bnhd& k, const mosaic_bnhd& v, const int64_t* idx,
          const int32_t* lens, int32_t batch, int32_t nq, int32_t nk, int32_t hq, int32_t hk, int32_t bs, int32_t K, float scale) {
    p.q = static_cast<const bf16_t*>(q.ptr); p.q_sb = q.stride_b; p.q_sn = q.stride_n; p.q_sh = q.stride_h;
    p.k = static_cast<const bf16_t*>(k.ptr); p.k_sb = k.stride_b; p.k_sn = k.stride_n; p.k_sh = k.stride_h;
    p.v = static_cast<const bf16_t*>(v.ptr); p.v_sb = v.stride_b; p.v_sn = v.stride_n; p.v_sh = v.stride_h;
    p.idx = idx; p.lens = lens;
    p.B = batch; p.Nq = nq; p.Nk = nk; p.Hq = hq; p.Hk = hk; p.G = hq / hk; p.QW = 16 / p.G; p.bs = bs; p.K = K;
    p.nb = (nk + bs - 1) / bs;
    p.qtiles = (nq + kWaves * p.QW - 1) / (kWaves * p.QW);
    p.splits = 1;
    p.scale = scale > 0.f ? scale : 0.125f;   // head_dim^-0.5
    p.c = p.scale * kLog2e;
}

int words_of(int32_t nq) { return (nq + kMarkTokens - 1) / kMarkTokens * kMarkWords; }

hipError_t launch(const void* fn, dim3 grid, void** args, hipStream_t s) { return hipLaunchKernel(fn, grid, dim3(kThreads), args, 0, s); }

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

size_t mosaic_query_attn_fwd_workspace_size(int32_t batch, int32_t num_queries, int32_t num_q_heads, int32_t num_kv_heads,
                                            int32_t block_count) {
    if (check_shape(batch, num_queries, 1, num_q_heads, num_kv_heads, kHeadDim, 64, block_count) != MOSAIC_OK) return 0;
    const int s = choose_split(batch, num_queries, num_q_heads, num_kv_heads, block_count);
    if (s == 1) return 0;
    const size_t rows = (size_t)batch * num_queries * num_q_heads;
    return up(s * rows * kHeadDim * sizeof(float)) + up(s * rows * sizeof(float2));
}

int mosaic_query_attn_fwd(mosaic_bnhd q, mosaic_bnhd k, mosaic_bnhd v, const int64_t* block_indices, const int32_t* kv_lens,
                          int32_t batch, int32_t num_queries, int32_t num_keys, int32_t num_q_heads, int32_t num_kv_heads,
                          int32_t head_dim, int32_t block_size, int32_t block_count, float softmax_scale, void* out, float* lse,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, head_dim, block_size, block_count)) return e;
    for (const mosaic_bnhd* t : {&q, &k, &v})
        if (int e = check_rows(*t)) return e;
    if (block_indices == nullptr || out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!aligned(block_indices, 8) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(kv_lens, 4)) return MOSAIC_ERR_ALIGNMENT;
    QueryAttnParams p{};
    fill(p, q, k, v, block_indices, kv_lens, batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count, softmax_scale);
    p.out = static_cast<bf16_t*>(out);
    p.lse = lse;
    p.splits = choose_split(batch, num_queries, num_q_heads, num_kv_heads, block_count);
    int64_t rows = (int64_t)batch * num_queries * num_q_heads;
    if (p.splits > 1) {
        const size_t need = mosaic_query_attn_fwd_workspace_size(batch, num_queries, num_q_heads, num_kv_heads, block_count);
        if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)) return MOSAIC_ERR_WORKSPACE;
        p.part_o = static_cast<float*>(workspace);
        p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + up(p.splits * rows * kHeadDim * sizeof(float)));
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    int total = p.qtiles * num_kv_heads * batch * p.splits;
    void* args[] = {&p, &total};
    if (launch((const void*)&query_attn_kernel, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (p.splits == 1) return MOSAIC_OK;
    void* jargs[] = {&p, &rows};
    return launch((const void*)&query_attn_join_kernel, dim3((unsigned)((rows + 15) / 16)), jargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

size_t mosaic_query_attn_bwd_workspace_size(int32_t batch, int32_t num_queries, int32_t num_keys, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t block_size) {
    if (check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, kHeadDim, block_size, 1) != MOSAIC_OK) return 0;
    const size_t rows = (size_t)batch * num_queries * num_q_heads, nb = ((size_t)num_keys + block_size - 1) / block_size;
    return 2 * up(rows * sizeof(float)) + up((size_t)batch * num_kv_heads * nb * words_of(num_queries) * sizeof(uint32_t));
}

int mosaic_query_attn_bwd(mosaic_bnhd q, mosaic_bnhd k, mosaic_bnhd v, const void* out, const float* lse, mosaic_bnhd grad_out,
                          const int64_t* block_indices, const int32_t* kv_lens, int32_t batch, int32_t num_queries,
                          int32_t num_keys, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                          int32_t block_count, float softmax_scale, void* grad_q, void* grad_k, void* grad_v, void* workspace,
                          size_t workspace_bytes, void* stream) {
    if (int e = check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, head_dim, block_size, block_count)) return e;
    for (const mosaic_bnhd* t : {&q, &k, &v, &grad_out})
        if (int e = check_rows(*t)) return e;
    if (!out || !lse || !block_indices || !grad_q || !grad_k || !grad_v) return MOSAIC_ERR_NULL_POINTER;
    for (const void* t : {out, (const void*)grad_q, (const void*)grad_k, (const void*)grad_v})
        if (!aligned(t, 16)) return MOSAIC_ERR_ALIGNMENT;
    if (!aligned(block_indices, 8) || !aligned(lse, 4) || !aligned(kv_lens, 4)) return MOSAIC_ERR_ALIGNMENT;
    const size_t need = mosaic_query_attn_bwd_workspace_size(batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)) return MOSAIC_ERR_WORKSPACE;
    QueryAttnParams p{};
    fill(p, q, k, v, block_indices, kv_lens, batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count, softmax_scale);
    p.go = static_cast<const bf16_t*>(grad_out.ptr);
    p.go_sb = grad_out.stride_b; p.go_sn = grad_out.stride_n; p.go_sh = grad_out.stride_h;
    p.o = static_cast<const bf16_t*>(out);
    p.lse = const_cast<float*>(lse);
    const size_t row_bytes = up((size_t)batch * num_queries * num_q_heads * sizeof(float));
    p.nlse = static_cast<float*>(workspace);
    p.ndelta = reinterpret_cast<float*>(static_cast<char*>(workspace) + row_bytes);
    p.marks = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + 2 * row_bytes);
    p.words = words_of(num_queries);
    p.out = static_cast<bf16_t*>(grad_q);
    p.dk = static_cast<bf16_t*>(grad_k);
    p.dv = static_cast<bf16_t*>(grad_v);
    const int64_t chunks = ((int64_t)p.nb + kUnion - 1) / kUnion;
    int groups = p.words / kMarkWords;
    if (chunks > 65535 || (double)groups * num_kv_heads * batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    int total = p.qtiles * num_kv_heads * batch;
    void* args[] = {&p, &total};
    if (launch((const void*)&query_attn_dq_kernel, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    void* margs[] = {&p, &groups};
    if (launch((const void*)&query_marks_kernel, dim3(groups * num_kv_heads * batch, (unsigned)chunks), margs, s) != hipSuccess)
        return MOSAIC_ERR_LAUNCH;
    int tiles = (num_keys + 63) / 64, dkv_total = tiles * num_kv_heads * batch;
    void* kargs[] = {&p, &tiles, &dkv_total};
    return launch((const void*)&query_attn_dkv_kernel, dim3(dkv_total), kargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
