// qattn.hip -- attention of query tokens over key blocks of their own, forward and backward (gfx950).
//
// Row (b, n, h) = query token n and kv head h, with K block indices (a set: an index counts once,
// one out of range not at all) and the G query heads of the group:
//   o = sum_u p_u v_u / l,  p_u = exp2(c q.k_u - m),  c = softmax_scale log2 e,  l = sum p_u
// over the keys u of the set's blocks, those past the sequence's length left out; a row without a
// key is zeros (lse -inf).  fp32 scores, maxima, sums and accumulators; P is rounded to bf16 for
// the PV product (an error of half a step of bf16 per term, as the output's own rounding).
//
// A workgroup takes 4 waves x QW = 32 / G tokens of one kv head, a wave the 32 rows (token, head) of
// its tokens.  The tokens' sets are united in LDS (a token mask per wave and block), and the union's
// blocks are staged once, 64 keys at a time, for all four waves; a wave skips the blocks none of its
// tokens has.  Neighbouring tokens of a mesh mostly choose the same blocks, so the union is little
// longer than one set (17.4 blocks for 32 tokens with 16 each on nside 64's field).  Tokens in no such
// order are taken in the order of a block of theirs (query_order_kernel): 10007 scattered points then
// unite 22 blocks instead of 313.
//
// Per tile of 64 keys, transposed so that a lane's scores are those of two rows
// (v_mfma_f32_32x32x16_bf16, a row in lanes r and r + 32):
//   S^T = K Q^T    A = K rows (16-byte LDS reads),  B = q (registers)
//   O^T = V^T P^T  A = V^T (transposing LDS reads), B = P, which S^T's accumulators already hold in
//                  operand order
// The reference m of a row moves only when a score exceeds it by 2^8; l sums the rounded P, so
// numerator and denominator share their roundings (the log-sum-exp, where one is asked for, sums P
// unrounded).  Rows that are no members of a block take P = 0, which leaves their accumulators' bits
// as they are: a row's result does not depend on who shares its wave.  Only 0 * NaN would, so where a
// workgroup ends with a value that is not finite it runs again, each product's accumulators restored
// for the rows that are no members, and what a row did not choose does not reach it then either.
//
// Bound by the vector ALU (exponentials, maxima, packing) beside the products, at three waves a SIMD:
// 49152 tokens with 12 query and 3 kv heads and 16 blocks of 64 keys (nside 64), 155 Gflop and 207 MB,
// take 231 us, 0.67 Pflop/s (a large matrix product reaches 1.2).  Each further block costs
// 11.4 us, and 57 us are spent before the first.  64 rows a wave (two waves a SIMD, half the LDS
// reads a score) measured 253 us there, 262 instead of 205 for two members' 10007 stations and 11.6
// instead of 9.4 for one token; 16 rows (v_mfma_f32_16x16x32_bf16) 345.
//
// Few queries: the union is split over workgroups and the partial (m, l, O) joined by a second
// kernel, or, where they have few keys too, a workgroup's waves share them (query_attn_few_kernel).
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "bsa_common.h"
#include "lds_dma.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32;          // rows (token, head) of a wave
constexpr int kTileElems = 64 * 64;
constexpr int kUnion = 1024;       // blocks whose members are marked at a time
constexpr int kMaxSplit = 32;
constexpr int kBuckets = 4096;     // of the order of tokens
constexpr float kTau = 8.f;        // a row's reference moves when a score exceeds it by 2^kTau

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
    float4* part_ml;           // [splits, rows] (m, l, l of the unrounded P, -)
    float* nlse;               // backward: -lse / c and -sum(o do) of each row
    float* ndelta;
    uint32_t* marks;           // backward: [B, Hk, nb, words] bit n: token n has the block
    int32_t* counts;           // backward: [B, Hk, nb] number of tokens of each block
    int32_t* starts;           // backward: [B, Hk, nb] where they begin in
    int32_t* takers;           // the tokens of each block, ascending
    int2* items;               // backward: (key tile, share | shares << 16) of each workgroup of grad k / v
    int32_t* slots;            // backward: [key tiles] first partial of a tile in several shares, else -1;
                               // then the number of items
    float* parts;              // backward: [slots, 2, 64 keys, 64] partials of grad k, grad v
    int share;                 // tokens of one share at most
    bf16_t* dk; bf16_t* dv;    // [B, Nk, Hk, 64]
    uint16_t* keys;            // [B, Hk, Nq] bucket of each token (null: tokens in their own order)
    int32_t* order;            // [B, Hk, Nq] tokens in the order they are taken in,
    int32_t* ordered;          // [B, Hk] where this is not 0
    int B, Nq, Nk, Hq, Hk, G, QW, bs, K, nb, words;
    int qtiles, splits;
    int qw_inverse;            // t / QW = t qw_inverse >> 16 for t < 256
    int short_rows;            // 64 rows of k and of v span less than 2^31 bytes (backward: and a sequence of q
                               // and of the output's gradient less than 2^32)
    float scale, c;
};

// LDS layout of 64-row tiles: 128-byte rows, 16-byte chunk c of row r at c ^ swz32(r).  Row reads
// (one chunk of 16 consecutive rows at a time) and transposing reads (four chunks of 4 rows) are
// both free of bank conflicts: over rows of one parity in 16 consecutive ones swz32 is a
// permutation of 0..7, and rows r and r + 2 of an aligned four differ in bit 2.
__device__ __forceinline__ int swz32(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

__device__ __forceinline__ bf16x8 tr_pair(const bf16_t* lo, const bf16_t* hi) {
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) v4i16*)(lo)));
    const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) v4i16*)(hi)));
    return as_bf16x8(make_uint4(a.x, a.y, b.x, b.y));
}

// Uses x, so that its load is waited for here.  A loop that counts direct-to-LDS loads itself has to
// begin without loads of the compiler's in flight: it would wait for them in every round, by a count
// that by then is that of the round's own loads, and the prefetch would overlap nothing.
__device__ __forceinline__ void arrived(bf16x8& x) {
    uint4 u = __builtin_bit_cast(uint4, x);
    asm volatile("" : "+v"(u.x), "+v"(u.y), "+v"(u.z), "+v"(u.w));
    x = as_bf16x8(u);
}

// The logical workgroup of a launched one: an XCD (workgroups go to the eight in turn) takes runs of
// 32 neighbours, which share key blocks in its L2, from all over the call, because sequences of a
// padded batch differ in work.  (One range of all the neighbours each, two sequences of 46209 and
// 44969 keys: 206 us instead of 183; runs of 8, 16, 64 and 128 are within 3 % of these there, and of
// each other where the work is even.)  The last, incomplete round keeps its order.
__device__ __forceinline__ int xcd_runs(int id, int total) {
    constexpr int kRun = 32;
    const int in = id & (8 * kRun - 1), first = id - in;
    return first + 8 * kRun > total ? id : first + (in & 7) * kRun + (in >> 3);
}

__device__ __forceinline__ int seq_keys(const QueryAttnParams& p, int b) {
    return p.lens == nullptr ? p.Nk : min(max(p.lens[b], 0), p.Nk);
}

// ------------------------------------------------------------------ the order of tokens
// Tokens of one kv head by a block of theirs: the one nearest the mean of them, in whatever order
// the row has them.  (10007 stations whose rows are in the order of scores: 22.0 blocks in a
// workgroup's union, as by the median; by the row's middle entry 31.7, by the mean itself 24.1.)

__device__ __forceinline__ int bucket_of(const QueryAttnParams& p, int blk) {
    return p.nb <= kBuckets ? blk : (int)((int64_t)blk * kBuckets / p.nb);
}

// Where the tokens' own order is already one of neighbours it is left as it is.  It is one if, of up to 64
// pairs of tokens that follow one another and have entries, at most a quarter have middle entries further apart than a 32nd
// of the blocks.  Every workgroup looks at the same pairs, then takes 32 tokens of one (b, h), eight lanes a
// token.  (49152 tokens that stay: 6 us, and 10 where each is read for it.)
constexpr int kKeyTokens = kThreads / 8;
__global__ __launch_bounds__(kThreads) void query_keys_kernel(QueryAttnParams p, int chunks) {
    const int bh = blockIdx.x / chunks, chunk = blockIdx.x - bh * chunks, h = bh % p.Hk, b = bh / p.Hk;
    const int tid = threadIdx.x, n0 = chunk * kKeyTokens, tokens = min(kKeyTokens, p.Nq - n0);
    const int pairs = min(64, p.Nq - 1);
    auto middle = [&](int n) {   // or, where that is no block, the first; -1: neither
        const int64_t* e = p.idx + (((int64_t)b * p.Nq + n) * p.Hk + h) * p.K;
        const int64_t x = e[p.K / 2], y = e[0];
        return x >= 0 && x < p.nb ? (int)x : y >= 0 && y < p.nb ? (int)y : -1;
    };
    bool both = false, apart = false;
    if (tid < pairs) {
        const int n = (int)((int64_t)tid * (p.Nq - 1) / pairs), x = middle(n), y = middle(n + 1);
        both = x >= 0 && y >= 0;
        apart = both && (int64_t)abs(x - y) * 32 > p.nb;
    }
    const bool sort = __syncthreads_count(apart) * 4 > __syncthreads_count(both);
    if (tid == 0 && chunk == 0) p.ordered[bh] = sort;
    if (!sort) return;
    const int64_t* e = p.idx + (((int64_t)b * p.Nq + n0 + min(tid >> 3, tokens - 1)) * p.Hk + h) * p.K;
    auto entry = [&](int i) {   // -1: none
        const int64_t blk = e[i];
        return blk >= 0 && blk < p.nb ? (int)blk : -1;
    };
    float sum = 0.f, count = 0.f;
    for (int i = tid & 7; i < p.K; i += 8) {
        const int blk = entry(i);
        sum += blk >= 0 ? (float)blk : 0.f;
        count += blk >= 0 ? 1.f : 0.f;
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        sum += __shfl_xor(sum, d);
        count += __shfl_xor(count, d);
    }
    const float mean = sum / count;
    float off = INFINITY;
    int nearest = -1;
    auto take = [&](float d, int blk) {
        const bool better = blk >= 0 && (d < off || (d == off && blk < nearest));
        off = better ? d : off;
        nearest = better ? blk : nearest;
    };
    for (int i = tid & 7; i < p.K; i += 8) {
        const int blk = entry(i);
        take(fabsf((float)blk - mean), blk);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        const float u = __shfl_xor(off, d);
        take(u, __shfl_xor(nearest, d));
    }
    if ((tid & 7) == 0 && tid >> 3 < tokens)
        p.keys[(int64_t)bh * p.Nq + n0 + (tid >> 3)] = (uint16_t)(nearest < 0 ? kBuckets : bucket_of(p, nearest));
}

// One workgroup = one (b, h): a counting sort by bucket.
// The order within a bucket is that of the LDS atomics; nothing depends on it.  (2 us where nothing is
// sorted; one workgroup's LDS atomics, and so linear in the tokens: 10 us for 10007, 37 for 49152, 130 for
// 196608, beside 89, 288 and 994 of the attention.)
constexpr int kOrderThreads = 1024, kOrderRun = 8;   // keys a thread has in flight
__global__ __launch_bounds__(kOrderThreads) void query_order_kernel(QueryAttnParams p) {
    if (p.ordered[blockIdx.x] == 0) return;
    __shared__ int start[kBuckets + 1];
    __shared__ int waves[kOrderThreads / 64];
    const int tid = threadIdx.x;
    for (int i = tid; i <= kBuckets; i += kOrderThreads) start[i] = 0;
    __syncthreads();
    const uint16_t* key = p.keys + (int64_t)blockIdx.x * p.Nq;
    int32_t* out = p.order + (int64_t)blockIdx.x * p.Nq;
    auto each = [&](auto use) {   // use(token, its key)
        for (int i0 = tid; i0 < p.Nq; i0 += kOrderThreads * kOrderRun) {
            int k[kOrderRun];
#pragma unroll
            for (int j = 0; j < kOrderRun; ++j) k[j] = key[min(i0 + j * kOrderThreads, p.Nq - 1)];
#pragma unroll
            for (int j = 0; j < kOrderRun; ++j)
                if (i0 + j * kOrderThreads < p.Nq) use(i0 + j * kOrderThreads, k[j]);
        }
    };
    each([&](int, int k) { atomicAdd(&start[k], 1); });
    __syncthreads();
    // exclusive prefix sums of the counts, 4 per thread; the last bucket is that of tokens without a block
    int c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = start[4 * tid + i];
        sum += c[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int x = __shfl_up(upto, d);
        upto += (tid & 63) >= d ? x : 0;
    }
    if ((tid & 63) == 63) waves[tid >> 6] = upto;
    __syncthreads();
    int at = upto - sum;
    for (int w = 0; w < tid >> 6; ++w) at += waves[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        start[4 * tid + i] = at;
        at += c[i];
    }
    if (tid == kOrderThreads - 1) start[kBuckets] = at;
    __syncthreads();
    each([&](int n, int k) { out[atomicAdd(&start[k], 1)] = n; });
}

// ------------------------------------------------------------------ tiles of a union

// LDS of the forward and grad-q kernels
struct RowsLds {
    __attribute__((aligned(1024))) bf16_t K[2][kTileElems];
    __attribute__((aligned(1024))) bf16_t V[2][kTileElems];
    __attribute__((aligned(16))) uint32_t members[kUnion][kWaves];   // bit t: token t of the wave has the block
    uint16_t list[kUnion];
    int tokens[kWaves * kRows];
    int found[kWaves];
};

// The workgroup's tokens (positions n0 .. of the order) into LDS; ends with a barrier.
__device__ __forceinline__ void load_tokens(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0) {
    const int64_t bh = (int64_t)b * p.Hk + h;
    const bool ordered = p.keys != nullptr && p.ordered[bh] != 0;
    for (int i = threadIdx.x; i < kWaves * p.QW; i += kThreads) {
        const int at = min(n0 + i, p.Nq - 1);
        L.tokens[i] = ordered ? p.order[bh * p.Nq + at] : at;
    }
    __syncthreads();
}

// Marks the members of blocks [c0, c0 + nc) among the workgroup's tokens and lists the blocks that
// have any, ascending; returns their number.  of_split < splits leaves other splits' blocks out
// (blocks u with u % splits == of_split remain).  Ends with a barrier.
__device__ __forceinline__ int unite(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, int end, int c0, int nc,
                                     int of_split, int splits) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < nc; i += kThreads) reinterpret_cast<uint4*>(L.members)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    // eight lanes a token
    const int tokens = min(kWaves * p.QW, p.Nq - n0);
    for (int t = tid >> 3; t < tokens; t += kThreads / 8) {
        const int64_t* e = p.idx + (((int64_t)b * p.Nq + L.tokens[t]) * p.Hk + h) * p.K;
        const int w = (t * p.qw_inverse) >> 16, of_wave = t - w * p.QW;
        const uint32_t bit = 1u << of_wave;
        for (int kk = tid & 7; kk < p.K; kk += 8) {
            const int64_t blk = e[kk] - c0;
            if (blk < 0 || blk >= nc) continue;
            const int u = c0 + (int)blk;
            if ((int64_t)u * p.bs < end && (splits == 1 || (uint32_t)u % (uint32_t)splits == (uint32_t)of_split))
                atomicOr(&L.members[blk][w], bit);
        }
    }
    __syncthreads();
    auto any = [&](int i) {
        if (i >= nc) return false;
        const uint4 x = *reinterpret_cast<const uint4*>(L.members[i]);
        return (x.x | x.y | x.z | x.w) != 0;
    };
    const int per = (nc + kThreads - 1) / kThreads * 64;   // blocks a wave lists
    int n = 0;
    for (int i = wave * per + lane; i - lane < (wave + 1) * per; i += 64)
        n += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(any(i)));
    if (lane == 0) L.found[wave] = n;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        at += w < wave ? L.found[w] : 0;
        total += L.found[w];
    }
    for (int i = wave * per + lane; i - lane < (wave + 1) * per; i += 64) {
        const bool on = any(i);
        const uint64_t m = __builtin_amdgcn_ballot_w64(on);
        if (on) L.list[at + (int)__builtin_popcountll(m & ((1ull << lane) - 1ull))] = (uint16_t)i;
        at += (int)__builtin_popcountll(m);
    }
    __syncthreads();
    return total;
}

// Runs `tile(K, V, members of this wave, valid keys)` over the tiles of this workgroup's share of
// the union, staged in two buffers with one barrier each.  Each wave loads 16 rows of K and V per
// tile: from a uniform base with per-lane offsets that do not change (64 rows within 2^31 bytes), or
// from 64-bit addresses, as the tile with the sequence's last key does, where the rows behind it
// repeat it (V's are zeroed: what P = 0 multiplies there).
template <typename Tile>
__device__ __forceinline__ void for_tiles(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, int split, int splits, Tile tile) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int end = seq_keys(p, b), sub = p.bs / 64;
    const bf16_t* kb = p.k + b * p.k_sb + h * p.k_sh;
    const bf16_t* vb = p.v + b * p.v_sb + h * p.v_sh;
    uint32_t ko[2], vo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 16 * wave + 8 * i + (lane >> 3), chunk = 8 * ((lane & 7) ^ swz32(row));
        ko[i] = 2u * (uint32_t)(row * p.k_sn + chunk);
        vo[i] = 2u * (uint32_t)(row * p.v_sn + chunk);
    }
    auto stage = [&](int key0, int buf) {
        if (p.short_rows && key0 + 64 <= end) {
            const bf16_t* kt = kb + (int64_t)key0 * p.k_sn;
            const bf16_t* vt = vb + (int64_t)key0 * p.v_sn;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                dma16(kt, ko[i], lds_addr(L.K[buf] + (16 * wave + 8 * i) * 64));
                dma16(vt, vo[i], lds_addr(L.V[buf] + (16 * wave + 8 * i) * 64));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 16 * wave + 8 * i + (lane >> 3), chunk = 8 * ((lane & 7) ^ swz32(row));
                const int64_t key = min(key0 + row, end - 1);
                dma16_at(kb + key * p.k_sn + chunk, lds_addr(L.K[buf] + (16 * wave + 8 * i) * 64));
                dma16_at(vb + key * p.v_sn + chunk, lds_addr(L.V[buf] + (16 * wave + 8 * i) * 64));
            }
        }
    };
    // without an order of tokens (few of them): shares by position in the list; else by block (see
    // unite), so that a row's share does not depend on the tokens beside it
    const bool by_block = p.keys != nullptr;
    const int live = min(p.nb, (int)((uint32_t)(end + p.bs - 1) / (uint32_t)p.bs));   // blocks with a key
    for (int c0 = 0; c0 < live; c0 += kUnion) {
        const int found = unite(p, L, b, h, n0, end, c0, min(kUnion, live - c0), split, by_block ? splits : 1);
        const int first = by_block ? 0 : (int)((uint32_t)(found * split) / (uint32_t)splits);
        const int past = by_block ? found : (int)((uint32_t)(found * (split + 1)) / (uint32_t)splits);
        for (int e0 = first; e0 < past; e0 += 64) {
            // up to 64 blocks of the list and this wave's members in registers: lane i holds block i
            const int count = min(64, past - e0);
            const int uv = L.list[e0 + min(lane, count - 1)];
            const int mv = (int)L.members[uv][wave];
            int key0 = (c0 + __builtin_amdgcn_readlane(uv, 0)) * p.bs, buf = 0;
            stage(key0, 0);
            for (int i = 0; i < count; ++i) {
                const uint32_t members = (uint32_t)__builtin_amdgcn_readlane(mv, i);
                for (int st = 0; st < sub; ++st) {
                    const bool more = st + 1 < sub ? key0 + 64 < end : i + 1 < count;
                    const int next = st + 1 < sub ? key0 + 64 : (c0 + __builtin_amdgcn_readlane(uv, min(i + 1, 63))) * p.bs;
                    wait_vmem();
                    lds_barrier();
                    if (more) stage(next, buf ^ 1);
                    const int valid = min(64, end - key0);
                    if (valid < 64) {
                        for (int z = threadIdx.x; z < (64 - valid) * 8; z += kThreads)
                            *reinterpret_cast<uint4*>(L.V[buf] + (valid + z / 8) * 64 + z % 8 * 8) = make_uint4(0, 0, 0, 0);
                        lds_barrier();
                    }
                    if (members != 0) tile(L.K[buf], L.V[buf], members, valid);
                    if (!more) break;   // past the last key, or past the list
                    key0 = next;
                    buf ^= 1;
                }
            }
            lds_barrier();   // the buffers are free for the next blocks
        }
        __syncthreads();     // and the lists
    }
}

// Per-lane LDS element offsets of the operand reads: row r, chunk 2 ds + hh, + 32 kt * 64; and the
// transposing reads of dims 32 dt + lane % 32, rows 4 hh + 0..3 and 8 more, + 16 rows * 64
struct TileReads {
    int row[4], tr[2][2];
    __device__ __forceinline__ void init(int lane) {
        const int r = lane & 31, hh = lane >> 5, s4 = lane & 15, half = (lane >> 4) & 1;
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) row[ds] = r * 64 + 8 * ((2 * ds + hh) ^ swz32(r));
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int sec = 0; sec < 2; ++sec) {
                const int rr = 4 * hh + (s4 >> 2) + 8 * sec;
                tr[dt][sec] = rr * 64 + 8 * ((4 * dt + 2 * half + ((s4 & 3) >> 1)) ^ swz32(rr)) + 4 * (s4 & 1);
            }
    }
    __device__ __forceinline__ bf16x8 rows(const bf16_t* T, int r0, int ds) const {
        return as_bf16x8(*reinterpret_cast<const uint4*>(T + r0 * 64 + row[ds]));
    }
    __device__ __forceinline__ bf16x8 cols(const bf16_t* T, int r0, int dt) const {
        return tr_pair(T + r0 * 64 + tr[dt][0], T + r0 * 64 + tr[dt][1]);
    }
};

__device__ __forceinline__ f32x16 splat(float x) {
    f32x16 y;
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = x;
    return y;
}

// acc + the 8 rounded values of one operand, two per instruction.  (A product with ones on the
// matrix pipe would do it too, but a 16-column one mixes rows r and r + 16, and zeros do not keep
// another row's NaN out.)
__device__ __forceinline__ float operand_sum(const bf16x8& x, float acc) {
    const uint4 u = __builtin_bit_cast(uint4, x);
    const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3f803f80u);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u.x), ones, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u.y), ones, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u.z), ones, acc, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u.w), ones, acc, false);
}

// Row r of a wave: token (position in the wave), query head, and its place in [B, Nq, Hq]
struct Row {
    int token, head;
    bool live;
    int64_t n, at;
    // tokens(i): the token at position n0 + i of the order
    template <typename Tokens>
    __device__ __forceinline__ void init(const QueryAttnParams& p, const Tokens& tokens, int b, int h, int n0, int wave, int r) {
        token = r / p.G;
        live = token < p.QW && n0 + wave * p.QW + token < p.Nq;
        head = h * p.G + (live ? r - token * p.G : 0);
        n = tokens(wave * p.QW + (live ? token : 0));
        at = ((int64_t)b * p.Nq + n) * p.Hq + head;
    }
    __device__ __forceinline__ bool in(uint32_t members) const { return live && (members >> token & 1); }
};

__device__ __forceinline__ void load_row(const bf16_t* x, int64_t sb, int64_t sn, int64_t sh, int b, const Row& r, int lane, bf16x8 (&f)[4]) {
    const bf16_t* at = x + b * sb + r.n * sn + r.head * sh + 8 * (lane >> 5);
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) f[ds] = as_bf16x8(ld16(at + 16 * ds));
}
__device__ __forceinline__ void arrived(bf16x8 (&f)[4]) {
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) arrived(f[ds]);
}

__device__ __forceinline__ void store_row(bf16_t* out, int64_t at, int lane, const f32x16 (&o)[2], float f) {
    bf16_t* d = out + at * 64 + 4 * (lane >> 5);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<uint2*>(d + 32 * dt + 8 * g4) = make_uint2(pack_bf16x2(o[dt][4 * g4] * f, o[dt][4 * g4 + 1] * f),
                                                                         pack_bf16x2(o[dt][4 * g4 + 2] * f, o[dt][4 * g4 + 3] * f));
}

// In a branch that is rarely taken: keeps the compiler from computing it always and selecting.
__device__ __forceinline__ void seldom() { asm volatile(""); }

// Scores of keys at or past `valid` become `fill` (accumulator element e of key half kt: key
// 32 kt + 8 (e / 4) + 4 hh + e % 4).  `valid` is opaque to the compiler, which would otherwise keep
// the comparisons of all calls in scalar registers at once.
__device__ __forceinline__ void mask_keys(f32x16& s, int kt, int hh, int valid, float fill) {
    int left = valid - 32 * kt - 4 * hh;
    asm volatile("" : "+v"(left));
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 8 * (e >> 2) + (e & 3) < left ? s[e] : fill;
}

struct FwdState {
    f32x16 o[2];      // O^T [dim tile]
    float m, l, lx;   // reference, and this lane's parts of the sums of the rounded and unrounded P
};

// One tile of 64 keys, keys(half, step) its A operands.  SAFE: the rows that are no members of it get
// their accumulators back after its products.
template <bool LSE, bool SAFE, typename Keys>
__device__ __forceinline__ void attend_tile(float c, const TileReads& tr, const Keys& keys, const bf16_t* Vt, const bf16x8 (&qf)[4],
                                            bool member, int valid, FwdState& a) {
    const int hh = (threadIdx.x & 63) >> 5;
    f32x16 s[2] = {splat(0.f), splat(0.f)};   // [key half]
    // operands are read two steps ahead (at this register count the compiler would otherwise read
    // each where it is used, and wait for it)
    bf16x8 k[4][2];
#pragma unroll
    for (int ds = 0; ds < 2; ++ds)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) k[ds][kt] = keys(kt, ds);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = mfma32(k[ds][kt], qf[ds], s[kt]);
        if (ds < 2) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) k[ds + 2][kt] = keys(kt, ds + 2);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (valid < 64) {
        seldom();
        mask_keys(s[0], 0, hh, valid, -INFINITY);
        mask_keys(s[1], 1, hh, valid, -INFINITY);
    }
    // (the maximum that NaN wins takes three operands and no canonicalising instruction)
    float mt = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) mt = __builtin_elementwise_maximum(mt, s[kt][e]);
    mt = xor32_max(mt) * c;
    const bool move = member && mt > a.m + kTau;
    if (__builtin_amdgcn_ballot_w64(move)) {   // rare after a row's first tile
        const float alpha = move ? __builtin_amdgcn_exp2f(a.m - mt) : 1.f;
        a.m = move ? mt : a.m;
        a.o[0] *= alpha;
        a.o[1] *= alpha;
        a.l *= alpha;
        if constexpr (LSE) a.lx *= alpha;
    }
    bf16x8 v[2];          // V^T of the first 16 keys: read before the exponentials
    if constexpr (!SAFE) {
        v[0] = tr.cols(Vt, 0, 0);
        v[1] = tr.cols(Vt, 0, 1);
    }
    const float ref = member ? a.m : INFINITY;   // P = 0 for the others
    bf16x8 pb[2][2];                             // [key half][16-key step]
    float lt[2] = {0.f, 0.f}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt][8 * s2 + 2 * i], c, -ref));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kt][8 * s2 + 2 * i + 1], c, -ref));
                if constexpr (LSE) sum[kt] += p0 + p1;
                w[i] = pack_bf16x2(p0, p1);
            }
            pb[kt][s2] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
            lt[kt] = operand_sum(pb[kt][s2], lt[kt]);
        }
    if (!SAFE || member) {
        a.l += lt[0] + lt[1];
        if constexpr (LSE) a.lx += sum[0] + sum[1];
    }
    if constexpr (SAFE) {
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
            f32x16 y = a.o[dt];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) y = mfma32(tr.cols(Vt, 32 * kt + 16 * s2, dt), pb[kt][s2], y);
            if (member) a.o[dt] = y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 next[2];
            if (j < 3)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) next[dt] = tr.cols(Vt, 16 * (j + 1), dt);
#pragma unroll
            for (int dt = 0; dt < 2; ++dt) a.o[dt] = mfma32(v[dt], pb[j >> 1][j & 1], a.o[dt]);
            if (j < 3) {
                v[0] = next[0];
                v[1] = next[1];
            }
        }
    }
}

__device__ __forceinline__ void clear(FwdState& a) {
    a.o[0] = a.o[1] = splat(0.f);
    a.m = -FLT_MAX;   // finite, so that keys whose score is -inf are exp2(-inf) = 0 also before any other
    a.l = a.lx = 0.f;
}

template <bool LSE, bool SAFE>
__device__ __forceinline__ void attend(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, int split, const Row& row,
                                       const bf16x8 (&qf)[4], FwdState& a) {
    TileReads tr;
    tr.init(threadIdx.x & 63);
    clear(a);
    for_tiles(p, L, b, h, n0, split, p.splits, [&](const bf16_t* Kt, const bf16_t* Vt, uint32_t members, int valid) {
        attend_tile<LSE, SAFE>(p.c, tr, [&](int kt, int ds) { return tr.rows(Kt, 32 * kt, ds); }, Vt, qf, row.in(members), valid, a);
    });
}

// Whether every element of x is finite (their difference with themselves is 0)
__device__ __forceinline__ bool finite(const f32x16& x) {
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) d = fmaf(0.f, x[e], d);
    return d == 0.f;
}

template <bool LSE>
__global__ __launch_bounds__(kThreads, 3) void query_attn_kernel(QueryAttnParams p, int total) {
    __shared__ RowsLds L;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_runs(blockIdx.x, total);
    const int split = id % p.splits, tile_id = id / p.splits % p.qtiles, rest = id / p.splits / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * kWaves * p.QW;
    load_tokens(p, L, b, h, n0);
    Row row;
    row.init(p, [&](int i) { return L.tokens[i]; }, b, h, n0, wave, lane & 31);
    bf16x8 qf[4];
    load_row(p.q, p.q_sb, p.q_sn, p.q_sh, b, row, lane, qf);
    arrived(qf);
    FwdState a;
    attend<LSE, false>(p, L, b, h, n0, split, row, qf, a);
    const bool ok = finite(a.o[0]) && finite(a.o[1]) && a.l - a.l == 0.f;
    if (__syncthreads_or(!ok)) attend<LSE, true>(p, L, b, h, n0, split, row, qf, a);
    const float l = xor32_add(a.l), lx = LSE ? xor32_add(a.lx) : 0.f;
    if (!row.live) return;
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.B * p.Nq * p.Hq;
        float* d = p.part_o + (split * rows + row.at) * 64 + 4 * hh;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4)
                *reinterpret_cast<float4*>(d + 32 * dt + 8 * g4) =
                    make_float4(a.o[dt][4 * g4], a.o[dt][4 * g4 + 1], a.o[dt][4 * g4 + 2], a.o[dt][4 * g4 + 3]);
        if (hh == 0) p.part_ml[split * rows + row.at] = make_float4(a.m, l, lx, 0.f);
        return;
    }
    // a row without a key, or with none whose score is above -inf, has l = 0 (any other at least 2^-8, or NaN)
    store_row(p.out, row.at, lane, a.o, l == 0.f ? 0.f : 1.f / l);
    if constexpr (LSE)
        if (hh == 0) p.lse[row.at] = a.m + __builtin_amdgcn_logf(lx);
}

// Joins the splits' partials: 16 lanes a row, 4 dims each.  Lane j holds the weights of splits j and
// j + 16, so that no load waits for another.
__global__ __launch_bounds__(kThreads) void query_attn_join_kernel(QueryAttnParams p, int64_t rows) {
    static_assert(kMaxSplit == 32, "two splits a lane");
    const int64_t at = (int64_t)blockIdx.x * 16 + threadIdx.x / 16, row = at < rows ? at : rows - 1;
    const int j = threadIdx.x % 16, d = 4 * j;
    float4 ml[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = j + 16 * i;
        ml[i] = s < p.splits ? p.part_ml[s * rows + row] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    }
    float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
    // l = 0: no key in that share (its m is the lowest value, as is that of one with nothing but NaN)
    float a[2], l = 0.f, lx = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        a[i] = ml[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - m);
        l = fmaf(a[i], ml[i].y, l);
        lx = fmaf(a[i], ml[i].z, lx);
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        l += __shfl_xor(l, x);
        lx += __shfl_xor(lx, x);
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int n = min(16, p.splits - 16 * i);
#pragma unroll 8
        for (int s = 0; s < n; ++s) {
            const float4 x = *reinterpret_cast<const float4*>(p.part_o + ((s + 16 * i) * rows + row) * 64 + d);
            const float w = __shfl(a[i], (threadIdx.x & 48) + s);
            o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
        }
    }
    if (at >= rows) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + row * 64 + d) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
    if (p.lse != nullptr && d == 0) p.lse[row] = m + __builtin_amdgcn_logf(lx);
}

// Few tokens with few keys, one token above all: one launch and no union in LDS.  A workgroup takes 32
// rows (32 / G tokens) and its waves the tiles of 64 keys in turn, each with its own accumulators; they
// are joined in LDS.  The tokens' entries, no more than 64, lie one in a lane of every wave.
//
// Bound by what one CU reads: 2048 keys (512 KB of k and v) take 14 us and half of them 9.4, where the
// union split over workgroups and its join take 16 and 11.5, and a launch more of the host (one token of
// 12 query and 3 kv heads, a call at a time: 15 and 19 us).  At 4096 keys it is 24 to 28 for 15 to 17, so
// kFewKeys is 2048.  100 tokens with 16 blocks of 64 and 16 heads to one: 15.5 for 34.  12 waves
// measured 5 % more, 16 spill (24 us), and tiles requested one ahead of their use the same.
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves, kFewKeys = 2048;

template <bool LSE>
__global__ __launch_bounds__(kFewThreads) void query_attn_few_kernel(QueryAttnParams p) {
    __shared__ __attribute__((aligned(1024))) bf16_t V[kFewWaves][kTileElems];   // a wave's tile, then its O
    __shared__ float4 ml[kFewWaves][kRows];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile_id = blockIdx.x % p.qtiles, rest = blockIdx.x / p.qtiles, h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * p.QW, entries = min(p.QW, p.Nq - n0) * p.K, end = seq_keys(p, b), sub = p.bs / 64;
    const bf16_t* kb = p.k + b * p.k_sb + h * p.k_sh;
    const bf16_t* vb = p.v + b * p.v_sb + h * p.v_sh;
    int blk = -1;
    if (lane < entries) {
        const int t = lane / p.K;
        const int64_t u = p.idx[(((int64_t)b * p.Nq + n0 + t) * p.Hk + h) * p.K + lane - t * p.K];
        blk = u >= 0 && u < p.nb && u * p.bs < end ? (int)u : -1;
    }
    Row row;
    row.init(p, [&](int i) { return n0 + i; }, b, h, n0, 0, r);
    bf16x8 qf[4];
    load_row(p.q, p.q_sb, p.q_sn, p.q_sh, b, row, lane, qf);
    // an entry's lane: the tokens with its block, and whether it is the first that names it
    uint32_t tokens = 0;
    bool first = blk >= 0;
    for (int j = 0, t = 0, of = 0; j < entries; ++j) {
        const bool same = __builtin_amdgcn_readlane(blk, j) == blk;
        tokens |= same ? 1u << t : 0u;
        first = first && !(same && j < lane);
        if (++of == p.K) {
            of = 0;
            ++t;
        }
    }
    const uint64_t firsts = __builtin_amdgcn_ballot_w64(first);
    const int rank = (int)__builtin_popcountll(firsts & ((1ull << lane) - 1ull)), units = (int)__builtin_popcountll(firsts) * sub;
    TileReads tr;
    tr.init(lane);
    FwdState a;
    auto walk = [&](auto safe) {
        clear(a);
        for (int u = wave; u < units; u += kFewWaves) {
            const int which = (int)((uint32_t)u / (uint32_t)sub);
            const int src = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(first && rank == which));
            const int key0 = __builtin_amdgcn_readlane(blk, src) * p.bs + (u - which * sub) * 64;
            if (key0 >= end) continue;
            const int valid = min(64, end - key0);
            bf16x8 k[2][4];   // rows past the end repeat the last one
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const bf16_t* kr = kb + (int64_t)min(key0 + 32 * kt + r, end - 1) * p.k_sn + 8 * hh;
#pragma unroll
                for (int ds = 0; ds < 4; ++ds) k[kt][ds] = as_bf16x8(ld16(kr + 16 * ds));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int vr = 8 * i + (lane >> 3), chunk = 8 * ((lane & 7) ^ swz32(vr));
                dma16_at(vb + (int64_t)min(key0 + vr, end - 1) * p.v_sn + chunk, lds_addr(V[wave] + 8 * i * 64));
            }
            wait_vmem();
            if (valid < 64)
                for (int z = lane; z < (64 - valid) * 8; z += 64)
                    *reinterpret_cast<uint4*>(V[wave] + (valid + z / 8) * 64 + z % 8 * 8) = make_uint4(0, 0, 0, 0);
            asm volatile("" ::: "memory");
            attend_tile<LSE, decltype(safe)::value>(p.c, tr, [&](int kt, int ds) { return k[kt][ds]; }, V[wave], qf,
                                                    row.in((uint32_t)__builtin_amdgcn_readlane((int)tokens, src)), valid, a);
            asm volatile("" ::: "memory");   // the tile is read before the next one, or O, takes its place
        }
    };
    walk(std::false_type{});
    const bool ok = finite(a.o[0]) && finite(a.o[1]) && a.l - a.l == 0.f;
    if (__builtin_amdgcn_ballot_w64(!ok)) walk(std::true_type{});   // (a wave by itself)
    float4* O = reinterpret_cast<float4*>(V[wave]);   // row r's dims 4 c .. at chunk c ^ (r % 16)
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            O[r * 16 + ((8 * dt + 2 * g4 + hh) ^ (r & 15))] = make_float4(a.o[dt][4 * g4], a.o[dt][4 * g4 + 1], a.o[dt][4 * g4 + 2], a.o[dt][4 * g4 + 3]);
    const float l = xor32_add(a.l), lx = LSE ? xor32_add(a.lx) : 0.f;
    if (hh == 0) ml[wave][r] = make_float4(a.m, l, lx, 0.f);
    __syncthreads();
    if (tid >= kRows * 16) return;
    // 16 threads a row
    Row to;
    to.init(p, [&](int i) { return n0 + i; }, b, h, n0, 0, tid / 16);
    if (!to.live) return;
    const int tr16 = tid / 16, c = tid % 16;
    float m = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) m = fmaxf(m, ml[w][tr16].x);
    float sum = 0.f, sumx = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
        const float4 part = ml[w][tr16], x = reinterpret_cast<const float4*>(V[w])[tr16 * 16 + (c ^ (tr16 & 15))];
        const float f = part.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(part.x - m);   // no key: its m is the lowest value
        sum = fmaf(f, part.y, sum);
        sumx = fmaf(f, part.z, sumx);
        o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(p.out + to.at * 64 + 4 * c) = make_uint2(pack_bf16x2(o.x * f, o.y * f), pack_bf16x2(o.z * f, o.w * f));
    if constexpr (LSE)
        if (c == 0) p.lse[to.at] = m + __builtin_amdgcn_logf(sumx);
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
//
// Bound as the forward, at two waves a SIMD (256 registers, nine more spilled, 40 bytes of scratch a lane):
// 116-121 us for 12288 tokens of 12 blocks, 16 query and 4 kv heads: 77 Gflop, 0.65 Pflop/s.
struct DqState {
    f32x16 dq[2], kbar[2];   // sum dS' k, sum P k [dim tile]
    float sum, rest;         // this lane's parts of sum dS' and of sum P (do.v - delta)
};

// SAFE as in the forward
template <bool SAFE>
__device__ __forceinline__ void differentiate(const QueryAttnParams& p, RowsLds& L, int b, int h, int n0, const Row& row,
                                              const bf16x8 (&qf)[4], const bf16x8 (&gf)[4], float nlse, float delta, DqState& a) {
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    TileReads tr;
    tr.init(lane);
    a.dq[0] = a.dq[1] = a.kbar[0] = a.kbar[1] = splat(0.f);
    a.sum = a.rest = 0.f;
    for_tiles(p, L, b, h, n0, 0, 1, [&](const bf16_t* Kt, const bf16_t* Vt, uint32_t members, int valid) {
        const bool member = row.in(members);
        const float off = member ? 0.f : -INFINITY;   // P = 0 and dS = 0 for the others
#pragma unroll 1
        for (int kt = 0; kt < 2; ++kt) {
            f32x16 s = splat(nlse), dp = splat(-delta);
            bf16x8 k[4], v[4];
#pragma unroll
            for (int ds = 0; ds < 2; ++ds) {
                k[ds] = tr.rows(Kt, 32 * kt, ds);
                v[ds] = tr.rows(Vt, 32 * kt, ds);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ds = 0; ds < 4; ++ds) {
                s = mfma32(k[ds], qf[ds], s);
                dp = mfma32(v[ds], gf[ds], dp);
                if (ds < 2) {
                    k[ds + 2] = tr.rows(Kt, 32 * kt, ds + 2);
                    v[ds + 2] = tr.rows(Vt, 32 * kt, ds + 2);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (valid < 64) {
                seldom();
                mask_keys(s, kt, hh, valid, -INFINITY);
                mask_keys(dp, kt, hh, valid, 0.f);
            }
            bf16x8 pb[2], db[2];
            float dsum = 0.f, rsum = 0.f;
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                uint32_t w[4], x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 8 * s2 + 2 * i;
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[e], p.c, off)), p1 = __builtin_amdgcn_exp2f(fmaf(s[e + 1], p.c, off));
                    const float d0 = p0 * dp[e], d1 = p1 * dp[e + 1];
                    dsum += d0 + d1;
                    w[i] = pack_bf16x2(p0, p1);
                    x[i] = pack_bf16x2(d0, d1);
                }
                pb[s2] = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
                db[s2] = as_bf16x8(make_uint4(x[0], x[1], x[2], x[3]));
                rsum = operand_sum(db[s2], rsum);
            }
            if (!SAFE || member) {
                a.sum += rsum;
                a.rest += dsum;
            }
            f32x16 dq[2] = {a.dq[0], a.dq[1]}, kbar[2] = {a.kbar[0], a.kbar[1]};
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) {
                    const bf16x8 kT = tr.cols(Kt, 32 * kt + 16 * s2, dt);
                    dq[dt] = mfma32(kT, db[s2], dq[dt]);
                    kbar[dt] = mfma32(kT, pb[s2], kbar[dt]);
                }
            if (!SAFE || member) {
                a.dq[0] = dq[0];
                a.dq[1] = dq[1];
                a.kbar[0] = kbar[0];
                a.kbar[1] = kbar[1];
            }
        }
    });
}

__global__ __launch_bounds__(kThreads, 2) void query_attn_dq_kernel(QueryAttnParams p, int total) {
    __shared__ RowsLds L;
    const int lane = threadIdx.x & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = xcd_runs(blockIdx.x, total);
    const int tile_id = id % p.qtiles, rest = id / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile_id * kWaves * p.QW;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (int64_t)p.B * p.Hk * p.nb; i += (int64_t)total * kThreads)
        p.counts[i] = 0;   // for query_marks_kernel
    load_tokens(p, L, b, h, n0);
    Row row;
    row.init(p, [&](int i) { return L.tokens[i]; }, b, h, n0, wave, lane & 31);
    bf16x8 qf[4], gf[4];
    load_row(p.q, p.q_sb, p.q_sn, p.q_sh, b, row, lane, qf);
    load_row(p.go, p.go_sb, p.go_sn, p.go_sh, b, row, lane, gf);
    float delta = 0.f;
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) {
        const uint4 ov = ld16(p.o + row.at * 64 + 16 * ds + 8 * hh), gv = __builtin_bit_cast(uint4, gf[ds]);
        const uint32_t ow[4] = {ov.x, ov.y, ov.z, ov.w}, gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) delta = fmaf(bf_lo(ow[i]), bf_lo(gw[i]), fmaf(bf_hi(ow[i]), bf_hi(gw[i]), delta));
    }
    delta = xor32_add(delta);
    const float lse = p.lse[row.at];
    float nlse = lse == -INFINITY ? 0.f : -lse / p.c;   // (nothing to add up for a row without a key)
    asm volatile("" : "+v"(nlse));
    arrived(qf);
    arrived(gf);
    DqState a;
    differentiate<false>(p, L, b, h, n0, row, qf, gf, nlse, delta, a);
    const bool ok = finite(a.dq[0]) && finite(a.dq[1]) && finite(a.kbar[0]) && finite(a.kbar[1]) && a.sum - a.sum == 0.f && a.rest - a.rest == 0.f;
    if (__syncthreads_or(!ok)) differentiate<true>(p, L, b, h, n0, row, qf, gf, nlse, delta, a);
    const float more = xor32_add(a.rest), sum = xor32_add(a.sum);
    if (!row.live) return;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) a.dq[dt][e] = fmaf(-sum, a.kbar[dt][e], a.dq[dt][e]);
    store_row(p.out, row.at, lane, a.dq, p.scale);
    if (hh == 0) {
        p.nlse[row.at] = nlse;
        p.ndelta[row.at] = -(delta + more);
    }
}

// The tokens of each block, as bits: a workgroup takes 512 tokens (16 words) of one kv head and up
// to kUnion blocks, marks in LDS and writes every word, so they need no clearing; the blocks' numbers
// of tokens are added up beside them (integers: their order does not matter).  7 us for 12288 tokens of
// 12 blocks in 4 heads (one entry at a time: 12).  A bit for every token and block: B Hk nb Nq / 8 bytes,
// 226 MB for one member of nside 128 with blocks of 64 and 3 kv heads, 16 times that at nside 256.
constexpr int kMarkTokens = 512, kMarkWords = kMarkTokens / 32;
__global__ __launch_bounds__(kThreads) void query_marks_kernel(QueryAttnParams p, int groups) {
    __shared__ __attribute__((aligned(16))) uint32_t bits[kUnion * kMarkWords];
    const int grp = blockIdx.x % groups, rest = blockIdx.x / groups;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int c0 = blockIdx.y * kUnion, nc = min(kUnion, p.nb - c0);
    for (int i = threadIdx.x; i < nc * kMarkWords; i += kThreads) bits[i] = 0;
    __syncthreads();
    const int n0 = grp * kMarkTokens, tokens = min(kMarkTokens, p.Nq - n0);
    // two lanes a token, eight entries of theirs at once (one seen twice does no harm)
    for (int t = threadIdx.x / 2; t < tokens; t += kThreads / 2) {
        const int64_t* e = p.idx + (((int64_t)b * p.Nq + n0 + t) * p.Hk + h) * p.K;
        for (int k0 = threadIdx.x % 2; k0 < p.K; k0 += 16) {
            int64_t blk[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) blk[j] = e[min(k0 + 2 * j, p.K - 1)] - c0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (blk[j] >= 0 && blk[j] < nc) atomicOr(&bits[blk[j] * kMarkWords + t / 32], 1u << (t % 32));
        }
    }
    __syncthreads();
    uint32_t* out = p.marks + (((int64_t)b * p.Hk + h) * p.nb + c0) * p.words + grp * kMarkWords;
    for (int i = threadIdx.x; i < nc * (kMarkWords / 4); i += kThreads) {
        const int blk = i / (kMarkWords / 4), w = i % (kMarkWords / 4) * 4;
        *reinterpret_cast<uint4*>(out + (int64_t)blk * p.words + w) = *reinterpret_cast<const uint4*>(bits + blk * kMarkWords + w);
    }
    int32_t* counts = p.counts + ((int64_t)b * p.Hk + h) * p.nb + c0;
    for (int i = threadIdx.x; i < nc; i += kThreads) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < kMarkWords; ++w) n += __builtin_popcount(bits[i * kMarkWords + w]);
        if (n > 0) atomicAdd(&counts[i], n);
    }
}

// Exclusive prefix sums over 1024 threads of a pair of counts, on top of `base`, which becomes the
// whole's.
__device__ __forceinline__ int2 prefix_1024(int2 x, int2& base, int2 (&sums)[16]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 y = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(y.x, d), v = __shfl_up(y.y, d);
        y.x += lane >= d ? u : 0;
        y.y += lane >= d ? v : 0;
    }
    if (lane == 63) sums[wave] = y;
    __syncthreads();
    int2 at = make_int2(base.x + y.x - x.x, base.y + y.y - x.y);
    for (int w = 0; w < 16; ++w) {
        at.x += w < wave ? sums[w].x : 0;
        at.y += w < wave ? sums[w].y : 0;
        base.x += sums[w].x;
        base.y += sums[w].y;
    }
    __syncthreads();
    return at;
}

// Where each block's tokens begin, and the workgroups of grad k / v: a tile of 64 keys whose block has
// more than p.share tokens is split into equal shares of them (blocks differ in popularity by
// factors: the most wanted one would run long after the others are done).  One workgroup; items are
// in the order of the tiles.
__global__ __launch_bounds__(1024) void query_plan_kernel(QueryAttnParams p, int tiles, int total) {
    __shared__ int2 sums[16];
    const int tid = threadIdx.x, blocks = p.B * p.Hk * p.nb;
    int2 base = make_int2(0, 0);
    for (int i0 = 0; i0 < blocks; i0 += 1024) {
        const int n = i0 + tid < blocks ? p.counts[i0 + tid] : 0;
        const int2 at = prefix_1024(make_int2(n, 0), base, sums);
        if (i0 + tid < blocks) p.starts[i0 + tid] = at.x;
    }
    base = make_int2(0, 0);
    for (int i0 = 0; i0 < total; i0 += 1024) {
        const int i = i0 + tid;
        int shares = 0;
        if (i < total) {
            const int kt = i % tiles, bh = i / tiles;
            const int count = p.counts[(int64_t)bh * p.nb + (int64_t)kt * 64 / p.bs];
            shares = max(1, (count + p.share - 1) / p.share);
        }
        const int2 at = prefix_1024(make_int2(shares, shares > 1 ? shares : 0), base, sums);   // items, partials
        for (int j = 0; j < shares; ++j) p.items[at.x + j] = make_int2(i, j | shares << 16);
        if (i < total) p.slots[i] = shares > 1 ? at.y : -1;
    }
    if (tid == 0) p.slots[total] = base.x;
}

// The tokens of each block, ascending, from its marks: one workgroup a block.
__global__ __launch_bounds__(kThreads) void query_takers_kernel(QueryAttnParams p) {
    __shared__ int sums[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int left = p.counts[blockIdx.x];
    if (left == 0) return;
    const uint32_t* marks = p.marks + (int64_t)blockIdx.x * p.words;
    int32_t* out = p.takers + p.starts[blockIdx.x];
    int seen = 0;
    for (int w0 = 0; w0 < p.words && seen < left; w0 += kThreads) {
        const uint32_t word = w0 + tid < p.words ? marks[w0 + tid] : 0;
        int upto = __builtin_popcount(word);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            upto += lane >= d ? x : 0;
        }
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        int at = seen + upto - __builtin_popcount(word);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            at += w < wave ? sums[w] : 0;
            seen += sums[w];
        }
        for (uint32_t m = word; m != 0; m &= m - 1) out[at++] = 32 * (w0 + tid) + __builtin_ctz(m);
        __syncthreads();
    }
}

// Sums of a split tile's partials, in the order of the shares (12288 tokens of 12 blocks in 4 heads: 10 us; row by row 12).
__global__ __launch_bounds__(kThreads) void query_sum_kernel(QueryAttnParams p, int tiles) {
    const int i = blockIdx.x, slot = p.slots[i];
    if (slot < 0) return;
    const int kt = i % tiles, bh = i / tiles, h = bh % p.Hk, b = bh / p.Hk;
    const int count = p.counts[(int64_t)bh * p.nb + (int64_t)kt * 64 / p.bs];
    const int shares = (count + p.share - 1) / p.share;
    // a thread: 4 dims of 8 rows of the 2 x 64, a share's loads in flight together
    constexpr int kEach = 128 * 16 / kThreads;
    const int d = threadIdx.x % 16 * 4, r0 = threadIdx.x / 16;
    float4 y[kEach] = {};
    for (int j = 0; j < shares; ++j) {
        const float* part = p.parts + ((int64_t)(slot + j) * 128 + r0) * 64 + d;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(part + i * (kThreads / 16) * 64);
            y[i].x += x.x; y[i].y += x.y; y[i].z += x.z; y[i].w += x.w;
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int r = r0 + i * (kThreads / 16), key = kt * 64 + r % 64;
        if (key >= p.Nk) continue;
        bf16_t* out = (r < 64 ? p.dk : p.dv) + (((int64_t)b * p.Nk + key) * p.Hk + h) * 64 + d;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(y[i].x, y[i].y), pack_bf16x2(y[i].z, y[i].w));
    }
}

// grad k, grad v.  One workgroup = 64 keys of one kv head and its share of the tokens that have the
// block: it walks them QS = 64 / G at a time (64 rows of q and do gathered straight into LDS).  Wave w = (key half w / 2,
// row half w % 2) forms S = q k^T and dP = do v^T of its 32 rows x 32 keys
// (v_mfma_f32_32x32x16_bf16); P and dS stay in registers as the B operands of dV^T += do^T P and
// dK^T += q^T dS, whose A operands are transposing LDS reads.  The row halves are added at the end.
//
// 120 us for 12288 tokens of 12 blocks, 16 query and 4 kv heads (77 Gflop): the gathers alone take
// about 56, the arithmetic alone 110.  Shares of three quarters of a block's mean; two slots instead
// of three and tokens read from the marks 147, tiles in no XCD's range 145, no shares 183.
constexpr int kListed = 2048;   // tokens listed at a time

struct KeysLds {
    __attribute__((aligned(1024))) bf16_t q[3][kTileElems];
    __attribute__((aligned(1024))) bf16_t g[3][kTileElems];
    float nlse[3][64], ndelta[3][64];
    int list[kListed];
};

// FINE: P and dS in two bf16 parts each, 16 bits, so that grad k and grad v are off by their own
// rounding alone (1.7e-3 in the 2-norm; with one part 2.3e-3, and 3.0e-3 for two tokens, whose terms
// may cancel).  Half as many products again (165 us for 120 above): for calls that are short anyway.
template <bool FINE>
__global__ __launch_bounds__(kThreads, 2) void query_attn_dkv_kernel(QueryAttnParams p, int tiles, int total) {
    __shared__ KeysLds L;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), kh = w >> 1, qh = w & 1;
    const int items = p.slots[total];
    if ((int)blockIdx.x >= items) return;
    const int2 item = p.items[xcd_remap(blockIdx.x, items)];   // (their work is even)
    const int kt = item.x % tiles, rest = item.x / tiles, h = rest % p.Hk, b = rest / p.Hk;
    const int share = item.y & 0xffff, shares = item.y >> 16;
    const int key0 = kt * 64, end = seq_keys(p, b);
    const int64_t all = p.counts[((int64_t)b * p.Hk + h) * p.nb + key0 / p.bs];
    const int from = (int)(all * share / shares), past = (int)(all * (share + 1) / shares);   // this share's tokens, by rank
    const int64_t block = ((int64_t)b * p.Hk + h) * p.nb + key0 / p.bs;
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
            arrived(kf);
            arrived(vf);
        }
        const bf16_t* qb = p.q + b * p.q_sb;
        const bf16_t* gb = p.go + b * p.go_sb;
        const float* nlse = p.nlse + (int64_t)b * p.Nq * p.Hq;
        const float* ndelta = p.ndelta + (int64_t)b * p.Nq * p.Hq;
        int64_t qoff[2], goff[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int chunk = 8 * ((lane & 7) ^ swz32(16 * w + 8 * i + (lane >> 3)));
            qoff[i] = lhead[i] * p.q_sh + chunk;
            goff[i] = lhead[i] * p.go_sh + chunk;
        }
        // Step s's rows into slot `buf`; entries past the list repeat its last one.  Six loads a wave,
        // whatever the step, so that waiting for all but the newest request is one count.  The tokens
        // of the step after it are read from the list meanwhile.
        int tok[3];
        auto look = [&](int s, int count) {
#pragma unroll
            for (int i = 0; i < 3; ++i) tok[i] = L.list[min(s * QS + ltok[i], count - 1)];
        };
        auto request = [&](int s, int buf, int count) {
            if (p.short_rows) {   // offsets from the tensors' starts fit 32 bits
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row0 = 16 * w + 8 * i;
                    dma16(qb, 2u * ((uint32_t)tok[i] * (uint32_t)p.q_sn + (uint32_t)qoff[i]), lds_addr(L.q[buf] + row0 * 64));
                    dma16(gb, 2u * ((uint32_t)tok[i] * (uint32_t)p.go_sn + (uint32_t)goff[i]), lds_addr(L.g[buf] + row0 * 64));
                }
                const uint32_t at = 4u * ((uint32_t)tok[2] * (uint32_t)p.Hq + (uint32_t)lhead[2]);
                if (lane < 16) {
                    dma4(nlse, at, lds_addr(L.nlse[buf] + 16 * w));
                    dma4(ndelta, at, lds_addr(L.ndelta[buf] + 16 * w));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row0 = 16 * w + 8 * i;
                    dma16_at(qb + (int64_t)tok[i] * p.q_sn + qoff[i], lds_addr(L.q[buf] + row0 * 64));
                    dma16_at(gb + (int64_t)tok[i] * p.go_sn + goff[i], lds_addr(L.g[buf] + row0 * 64));
                }
                const int64_t at = (int64_t)tok[2] * p.Hq + lhead[2];
                if (lane < 16) {
                    dma4_at(nlse + at, lds_addr(L.nlse[buf] + 16 * w));
                    dma4_at(ndelta + at, lds_addr(L.ndelta[buf] + 16 * w));
                }
            }
            look(s + 1, count);
        };
        auto tr_read = [&](const bf16_t* T, int q0, int dt) { return tr_pair(T + q0 * 64 + tr[dt][0], T + q0 * 64 + tr[dt][1]); };
        auto step = [&](int buf, int rows) {
            const bf16_t* Qc = L.q[buf];
            const bf16_t* Gc = L.g[buf];
            // reads are ahead of their products and exponentials throughout (the compiler left to itself
            // waits for each)
            f32x16 s, dp;
            bf16x8 qa[4], ga[4];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                qa[kk] = as_bf16x8(*reinterpret_cast<const uint4*>(Qc + 32 * qh * 64 + rd[kk]));
                ga[kk] = as_bf16x8(*reinterpret_cast<const uint4*>(Gc + 32 * qh * 64 + rd[kk]));
            }
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const float4 l4 = *reinterpret_cast<const float4*>(L.nlse[buf] + 32 * qh + 8 * g4 + 4 * hh);
                const float4 d4 = *reinterpret_cast<const float4*>(L.ndelta[buf] + 32 * qh + 8 * g4 + 4 * hh);
                s[4 * g4] = l4.x; s[4 * g4 + 1] = l4.y; s[4 * g4 + 2] = l4.z; s[4 * g4 + 3] = l4.w;
                dp[4 * g4] = d4.x; dp[4 * g4 + 1] = d4.y; dp[4 * g4 + 2] = d4.z; dp[4 * g4 + 3] = d4.w;
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                s = mfma32(qa[kk], kf[kk], s);
                dp = mfma32(ga[kk], vf[kk], dp);
                if (kk < 2) {
                    qa[kk + 2] = as_bf16x8(*reinterpret_cast<const uint4*>(Qc + 32 * qh * 64 + rd[kk + 2]));
                    ga[kk + 2] = as_bf16x8(*reinterpret_cast<const uint4*>(Gc + 32 * qh * 64 + rd[kk + 2]));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (rows < 64) {   // rows past the list, or past QS G: P = 0 and dS = 0
                seldom();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool on = 32 * qh + 8 * (e >> 2) + 4 * hh + (e & 3) < rows;
                    s[e] = on ? s[e] : -INFINITY;
                    dp[e] = on ? dp[e] : 0.f;
                }
            }
            bf16x8 gT[2][2], qT[2][2];   // [dim tile][16 rows]
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) gT[dt][ch] = tr_read(Gc, 32 * qh + 16 * ch, dt);
            __builtin_amdgcn_sched_barrier(0);
            bf16x8 pb[2], db[2], pl[2], dl[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float pr = __builtin_amdgcn_exp2f(s[e] * p.c), ds = pr * dp[e];
                pb[e >> 3][e & 7] = (__bf16)pr;
                db[e >> 3][e & 7] = (__bf16)ds;
                if constexpr (FINE) {
                    pl[e >> 3][e & 7] = (__bf16)(pr - (float)pb[e >> 3][e & 7]);
                    dl[e >> 3][e & 7] = (__bf16)(ds - (float)db[e >> 3][e & 7]);
                }
            }
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int ch = 0; ch < 2; ++ch) qT[dt][ch] = tr_read(Qc, 32 * qh + 16 * ch, dt);
#pragma unroll
            for (int ch = 0; ch < 2; ++ch)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) {
                    dvT[dt] = mfma32(gT[dt][ch], pb[ch], dvT[dt]);
                    if constexpr (FINE) dvT[dt] = mfma32(gT[dt][ch], pl[ch], dvT[dt]);
                }
#pragma unroll
            for (int ch = 0; ch < 2; ++ch)
#pragma unroll
                for (int dt = 0; dt < 2; ++dt) {
                    dkT[dt] = mfma32(qT[dt][ch], db[ch], dkT[dt]);
                    if constexpr (FINE) dkT[dt] = mfma32(qT[dt][ch], dl[ch], dkT[dt]);
                }
        };
        const int32_t* takers = p.takers + p.starts[block];
        const int run = kListed / QS * QS;   // tokens listed at a time
        for (int c0 = from; c0 < past; c0 += run) {
            const int count = min(run, past - c0), steps = (count + QS - 1) / QS;
            for (int i = tid; i < count; i += kThreads) L.list[i] = takers[c0 + i];
            __syncthreads();
            // a ring of three slots: a step's rows are requested two steps before it
            look(0, count);
            request(0, 0, count);
            request(1, 1, count);
            for (int s = 0, buf = 0; s < steps; ++s) {
                asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
                lds_barrier();
                request(s + 2, buf == 0 ? 2 : buf - 1, count);
                step(buf, min(QS, count - s * QS) * p.G);
                buf = buf == 2 ? 0 : buf + 1;
            }
            wait_vmem();
            __syncthreads();
        }
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
    if (shares > 1) {
        if (qh == 0) {   // rows past the sequence's end too: zeros
            float* d = p.parts + ((int64_t)(p.slots[item.x] + share) * 128 + 32 * kh + r) * 64 + 4 * hh;
            const bool on = key < end;
#pragma unroll
            for (int dt = 0; dt < 2; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const f32x16 &x = dkT[dt], &y = dvT[dt];
                    *reinterpret_cast<float4*>(d + 32 * dt + 8 * g4) =
                        on ? make_float4(x[4 * g4] * p.scale, x[4 * g4 + 1] * p.scale, x[4 * g4 + 2] * p.scale, x[4 * g4 + 3] * p.scale) : make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4*>(d + 64 * 64 + 32 * dt + 8 * g4) =
                        on ? make_float4(y[4 * g4], y[4 * g4 + 1], y[4 * g4 + 2], y[4 * g4 + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
        }
        return;
    }
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
    const int64_t per = kWaves * (kRows / (hq / hk)), tiles = ((int64_t)nq + per - 1) / per;
    if ((double)tiles * hk * batch * kMaxSplit > 2147483647.0) return MOSAIC_ERR_SHAPE;
    if ((double)((nk + 63) / 64) * hk * batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    if (((double)nq / kKeyTokens + 1) * hk * batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    return MOSAIC_OK;
}

// fp32 carries the scale and its reciprocal, times the logarithms that the backward divides by it.
bool scale_ok(float scale) { return scale <= 0.f || (scale >= 1e-30f && scale <= 1e30f); }

// Workgroups where the union is in one piece.
int64_t groups_of(int32_t batch, int32_t nq, int32_t hq, int32_t hk) {
    const int64_t per = kWaves * (kRows / (hq / hk));
    return (nq + per - 1) / per * hk * batch;
}
// Shares of the union: below one workgroup per CU it is split, up to two per CU together.
int choose_split(int32_t batch, int32_t nq, int32_t hq, int32_t hk, int32_t K) {
    const int64_t wgs = groups_of(batch, nq, hq, hk);
    if (wgs >= 256) return 1;
    const int64_t s = 512 / wgs;
    return (int)(s < K ? (s < kMaxSplit ? s : kMaxSplit) : (K < kMaxSplit ? K : kMaxSplit));
}

// Whether the call is one of query_attn_few_kernel: few workgroups, whose tokens name few keys each.
bool few(int32_t batch, int32_t nq, int32_t hq, int32_t hk, int32_t bs, int32_t K) {
    const int64_t tokens = nq < kRows / (hq / hk) ? nq : kRows / (hq / hk), entries = tokens * K;
    return groups_of(batch, nq, hq, hk) < 256 && entries <= 64 && entries * bs <= kFewKeys;
}

// Whether tokens may be taken in another order: with more than one workgroup of them.
bool may_order(int32_t nq, int32_t hq, int32_t hk) { return nq > kWaves * (kRows / (hq / hk)); }
int key_chunks(int32_t nq) { return (nq + kKeyTokens - 1) / kKeyTokens; }
size_t order_bytes(int32_t batch, int32_t nq, int32_t hq, int32_t hk) {
    if (!may_order(nq, hq, hk)) return 0;
    const size_t rows = (size_t)batch * hk * nq;
    return up(rows * sizeof(uint16_t)) + up(rows * sizeof(int32_t)) + up((size_t)batch * hk * sizeof(int32_t));
}
// Bytes of the forward's partials, behind which its workspace holds the order.
size_t part_bytes(int32_t batch, int32_t nq, int32_t hq, int32_t hk, int32_t K) {
    const int s = choose_split(batch, nq, hq, hk, K);
    const size_t rows = s == 1 ? 0 : (size_t)batch * nq * hq;
    return up(s * rows * kHeadDim * sizeof(float)) + up(s * rows * sizeof(float4));
}
void place_order(QueryAttnParams& p, char* ws) {
    if (!may_order(p.Nq, p.Hq, p.Hk)) return;
    const size_t rows = (size_t)p.B * p.Hk * p.Nq;
    p.keys = reinterpret_cast<uint16_t*>(ws);
    p.order = reinterpret_cast<int32_t*>(ws + up(rows * sizeof(uint16_t)));
    p.ordered = reinterpret_cast<int32_t*>(ws + up(rows * sizeof(uint16_t)) + up(rows * sizeof(int32_t)));
}

void fill(QueryAttnParams& p, const mosaic_bnhd& q, const mosaic_bnhd& k, const mosaic_bnhd& v, const int64_t* idx,
          const int32_t* lens, int32_t batch, int32_t nq, int32_t nk, int32_t hq, int32_t hk, int32_t bs, int32_t K, float scale, int rows) {
    p.q = static_cast<const bf16_t*>(q.ptr); p.q_sb = q.stride_b; p.q_sn = q.stride_n; p.q_sh = q.stride_h;
    p.k = static_cast<const bf16_t*>(k.ptr); p.k_sb = k.stride_b; p.k_sn = k.stride_n; p.k_sh = k.stride_h;
    p.v = static_cast<const bf16_t*>(v.ptr); p.v_sb = v.stride_b; p.v_sn = v.stride_n; p.v_sh = v.stride_h;
    p.idx = idx; p.lens = lens;
    p.B = batch; p.Nq = nq; p.Nk = nk; p.Hq = hq; p.Hk = hk; p.G = hq / hk; p.QW = rows / p.G; p.bs = bs; p.K = K;
    p.nb = (nk + bs - 1) / bs;
    p.qtiles = (nq + kWaves * p.QW - 1) / (kWaves * p.QW);
    p.splits = 1;
    p.qw_inverse = (65536 + p.QW - 1) / p.QW;
    const int64_t most = (int64_t)1 << 23;   // 64 rows of 2^23 bf16 are 2^30 bytes
    p.short_rows = k.stride_n >= 0 && k.stride_n <= most && v.stride_n >= 0 && v.stride_n <= most;
    p.scale = scale > 0.f ? scale : 0.125f;   // head_dim^-0.5
    p.c = p.scale * kLog2e;
}

int words_of(int32_t nq) { return (nq + kMarkTokens - 1) / kMarkTokens * kMarkWords; }

hipError_t launch(const void* fn, dim3 grid, void** args, hipStream_t s, int threads = kThreads) {
    return hipLaunchKernel(fn, grid, dim3(threads), args, 0, s);
}

// Workspace of the backward, and the tokens of one share of a key tile: three quarters of what a block
// has on average (grad k / v and the sums at 12288 tokens of nside 32: 133 us, with half as many again
// 139), fewer where the tiles alone do not fill the chip twice.  Where there are many tiles only those that would
// outlast the others are split: a share is a kShares-th of the call at least (a quarter of what a resident
// workgroup does), so the partials stay below 2 kShares tiles, 128 MiB, however large the call.  (A training
// step of four members of nside 64, 16 blocks of 64: 4.14-4.20 ms and 240 MiB, in shares of three quarters of a
// mean 4.23-4.30 ms and 880 MiB; one of nside 128 4.5 ms either way, 402 MiB for 1042.)
constexpr int64_t kShares = 2048;
struct BwdLayout {
    size_t nlse, ndelta, marks, counts, starts, takers, plan, slots, parts, order, bytes;
    int64_t items;   // workgroups of grad k / v at most
    int64_t pairs;   // (token, block) pairs at most
    int share;
};
BwdLayout bwd_layout(int32_t batch, int32_t nq, int32_t nk, int32_t hq, int32_t hk, int32_t bs, int32_t K) {
    BwdLayout a{};
    const int64_t nb = ((int64_t)nk + bs - 1) / bs, tiles = ((int64_t)nk + 63) / 64 * hk * batch;
    const int64_t chosen = (int64_t)nq * (K < nb ? K : nb);                // (token, block) pairs of a kv head at most
    const int64_t pairs = chosen * hk * batch * (bs / 64);                 // (token, key tile)
    int64_t share = chosen / nb * 3 / 4;
    if (tiles < 512 && share > pairs / 512) share = pairs / 512;
    if (share < pairs / kShares) share = pairs / kShares;
    if (share < 64) share = 64;
    if (share < (nq + 4095) / 4096) share = (nq + 4095) / 4096;            // a tile's shares are counted in 16 bits
    a.share = (int)(share < 0x7fffffff ? share : 0x7fffffff);
    // a tile with c tokens has at most 1 + c / share shares, of one with several there are 2 c / share at most
    a.items = tiles + pairs / a.share;
    a.pairs = chosen * hk * batch;
    const int64_t slots = 2 * (pairs / a.share) + 2;
    const size_t rows = up((size_t)batch * nq * hq * sizeof(float));
    a.ndelta = a.nlse + rows;
    a.marks = a.ndelta + rows;
    a.counts = a.marks + up((size_t)batch * hk * nb * words_of(nq) * sizeof(uint32_t));
    a.starts = a.counts + up((size_t)batch * hk * nb * sizeof(int32_t));
    a.takers = a.starts + up((size_t)batch * hk * nb * sizeof(int32_t));
    a.plan = a.takers + up((size_t)batch * hk * chosen * sizeof(int32_t));
    a.slots = a.plan + up((size_t)a.items * sizeof(int2));
    a.parts = a.slots + up((size_t)(tiles + 1) * sizeof(int32_t));
    a.order = a.parts + up((size_t)slots * 128 * kHeadDim * sizeof(float));
    a.bytes = a.order + order_bytes(batch, nq, hq, hk);
    return a;
}

int launch_order(QueryAttnParams& p, hipStream_t s) {
    if (p.keys == nullptr) return MOSAIC_OK;
    int chunks = key_chunks(p.Nq);
    void* args[] = {&p, &chunks};
    if (launch((const void*)&query_keys_kernel, dim3(p.B * p.Hk * chunks), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    return launch((const void*)&query_order_kernel, dim3(p.B * p.Hk), args, s, kOrderThreads) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

size_t mosaic_query_attn_fwd_workspace_size(int32_t batch, int32_t num_queries, int32_t num_q_heads, int32_t num_kv_heads,
                                            int32_t block_size, int32_t block_count) {
    if (check_shape(batch, num_queries, 1, num_q_heads, num_kv_heads, kHeadDim, block_size, block_count) != MOSAIC_OK) return 0;
    if (few(batch, num_queries, num_q_heads, num_kv_heads, block_size, block_count)) return 0;
    return part_bytes(batch, num_queries, num_q_heads, num_kv_heads, block_count) +
           order_bytes(batch, num_queries, num_q_heads, num_kv_heads);
}

int mosaic_query_attn_fwd(mosaic_bnhd q, mosaic_bnhd k, mosaic_bnhd v, const int64_t* block_indices, const int32_t* kv_lens,
                          int32_t batch, int32_t num_queries, int32_t num_keys, int32_t num_q_heads, int32_t num_kv_heads,
                          int32_t head_dim, int32_t block_size, int32_t block_count, float softmax_scale, void* out, float* lse,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, head_dim, block_size, block_count)) return e;
    if (!scale_ok(softmax_scale)) return MOSAIC_ERR_UNSUPPORTED;
    for (const mosaic_bnhd* t : {&q, &k, &v})
        if (int e = check_rows(*t)) return e;
    if (block_indices == nullptr || out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!aligned(block_indices, 8) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(kv_lens, 4)) return MOSAIC_ERR_ALIGNMENT;
    QueryAttnParams p{};
    fill(p, q, k, v, block_indices, kv_lens, batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count, softmax_scale, kRows);
    p.out = static_cast<bf16_t*>(out);
    p.lse = lse;
    p.splits = choose_split(batch, num_queries, num_q_heads, num_kv_heads, block_count);
    int64_t rows = (int64_t)batch * num_queries * num_q_heads;
    const size_t need = mosaic_query_attn_fwd_workspace_size(batch, num_queries, num_q_heads, num_kv_heads, block_size, block_count);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256))) return MOSAIC_ERR_WORKSPACE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (few(batch, num_queries, num_q_heads, num_kv_heads, block_size, block_count)) {
        p.qtiles = (num_queries + p.QW - 1) / p.QW;
        void* args[] = {&p};
        const void* fn = lse != nullptr ? (const void*)&query_attn_few_kernel<true> : (const void*)&query_attn_few_kernel<false>;
        return launch(fn, dim3((unsigned)(p.qtiles * num_kv_heads * batch)), args, s, kFewThreads) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
    }
    char* ws = static_cast<char*>(workspace);
    if (p.splits > 1) {
        p.part_o = reinterpret_cast<float*>(ws);
        p.part_ml = reinterpret_cast<float4*>(ws + up(p.splits * rows * kHeadDim * sizeof(float)));
    }
    place_order(p, ws + part_bytes(batch, num_queries, num_q_heads, num_kv_heads, block_count));
    if (int e = launch_order(p, s)) return e;
    int total = p.qtiles * num_kv_heads * batch * p.splits;
    void* args[] = {&p, &total};
    const void* fn = lse != nullptr ? (const void*)&query_attn_kernel<true> : (const void*)&query_attn_kernel<false>;
    if (launch(fn, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (p.splits == 1) return MOSAIC_OK;
    void* jargs[] = {&p, &rows};
    return launch((const void*)&query_attn_join_kernel, dim3((unsigned)((rows + 15) / 16)), jargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

size_t mosaic_query_attn_bwd_workspace_size(int32_t batch, int32_t num_queries, int32_t num_keys, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t block_size, int32_t block_count) {
    if (check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, kHeadDim, block_size, block_count) != MOSAIC_OK) return 0;
    return bwd_layout(batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count).bytes;
}

int mosaic_query_attn_bwd(mosaic_bnhd q, mosaic_bnhd k, mosaic_bnhd v, const void* out, const float* lse, mosaic_bnhd grad_out,
                          const int64_t* block_indices, const int32_t* kv_lens, int32_t batch, int32_t num_queries,
                          int32_t num_keys, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                          int32_t block_count, float softmax_scale, const void* fwd_workspace, void* grad_q, void* grad_k,
                          void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_shape(batch, num_queries, num_keys, num_q_heads, num_kv_heads, head_dim, block_size, block_count)) return e;
    if (!scale_ok(softmax_scale)) return MOSAIC_ERR_UNSUPPORTED;
    for (const mosaic_bnhd* t : {&q, &k, &v, &grad_out})
        if (int e = check_rows(*t)) return e;
    if (!out || !lse || !block_indices || !grad_q || !grad_k || !grad_v) return MOSAIC_ERR_NULL_POINTER;
    for (const void* t : {out, (const void*)grad_q, (const void*)grad_k, (const void*)grad_v})
        if (!aligned(t, 16)) return MOSAIC_ERR_ALIGNMENT;
    if (!aligned(block_indices, 8) || !aligned(lse, 4) || !aligned(kv_lens, 4) || !aligned(fwd_workspace, 256)) return MOSAIC_ERR_ALIGNMENT;
    const BwdLayout at = bwd_layout(batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count);
    if (workspace == nullptr || workspace_bytes < at.bytes || !aligned(workspace, 256)) return MOSAIC_ERR_WORKSPACE;
    // token lists are indexed in 31 bits
    if (at.items > 0x7fffffff || at.pairs > 0x7fffffff) return MOSAIC_ERR_SHAPE;
    QueryAttnParams p{};
    fill(p, q, k, v, block_indices, kv_lens, batch, num_queries, num_keys, num_q_heads, num_kv_heads, block_size, block_count, softmax_scale, kRows);
    p.go = static_cast<const bf16_t*>(grad_out.ptr);
    p.go_sb = grad_out.stride_b; p.go_sn = grad_out.stride_n; p.go_sh = grad_out.stride_h;
    auto spans = [&](const mosaic_bnhd& t) {   // a sequence's rows lie within 2^32 bytes of its first
        return t.stride_n >= 0 && t.stride_h >= 0 &&
               (double)(num_queries - 1) * t.stride_n + (double)(num_q_heads - 1) * t.stride_h + 64 < 2147483648.0;
    };
    p.short_rows = p.short_rows && spans(q) && spans(grad_out) && (double)num_queries * num_q_heads < 1073741824.0;
    p.o = static_cast<const bf16_t*>(out);
    p.lse = const_cast<float*>(lse);
    char* ws = static_cast<char*>(workspace);
    p.nlse = reinterpret_cast<float*>(ws + at.nlse);
    p.ndelta = reinterpret_cast<float*>(ws + at.ndelta);
    p.marks = reinterpret_cast<uint32_t*>(ws + at.marks);
    p.counts = reinterpret_cast<int32_t*>(ws + at.counts);
    p.starts = reinterpret_cast<int32_t*>(ws + at.starts);
    p.takers = reinterpret_cast<int32_t*>(ws + at.takers);
    p.items = reinterpret_cast<int2*>(ws + at.plan);
    p.slots = reinterpret_cast<int32_t*>(ws + at.slots);
    p.parts = reinterpret_cast<float*>(ws + at.parts);
    p.share = at.share;
    p.words = words_of(num_queries);
    // the forward's order, where it made one
    const bool have = fwd_workspace != nullptr && !few(batch, num_queries, num_q_heads, num_kv_heads, block_size, block_count);
    place_order(p, have ? static_cast<char*>(const_cast<void*>(fwd_workspace)) +
                              part_bytes(batch, num_queries, num_q_heads, num_kv_heads, block_count)
                        : ws + at.order);
    p.out = static_cast<bf16_t*>(grad_q);
    p.dk = static_cast<bf16_t*>(grad_k);
    p.dv = static_cast<bf16_t*>(grad_v);
    const int64_t chunks = ((int64_t)p.nb + kUnion - 1) / kUnion;
    int groups = p.words / kMarkWords;
    if (chunks > 65535 || (double)groups * num_kv_heads * batch > 2147483647.0) return MOSAIC_ERR_SHAPE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!have)
        if (int e = launch_order(p, s)) return e;
    int total = p.qtiles * num_kv_heads * batch;
    void* args[] = {&p, &total};
    if (launch((const void*)&query_attn_dq_kernel, dim3(total), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    void* margs[] = {&p, &groups};
    if (launch((const void*)&query_marks_kernel, dim3(groups * num_kv_heads * batch, (unsigned)chunks), margs, s) != hipSuccess)
        return MOSAIC_ERR_LAUNCH;
    int tiles = (num_keys + 63) / 64, key_tiles = tiles * num_kv_heads * batch;
    void* kargs[] = {&p, &tiles, &key_tiles};
    if (launch((const void*)&query_plan_kernel, dim3(1), kargs, s, 1024) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    void* targs[] = {&p};
    if (launch((const void*)&query_takers_kernel, dim3((unsigned)(p.nb * num_kv_heads * batch)), targs, s) != hipSuccess)
        return MOSAIC_ERR_LAUNCH;
    // rows of the steps in all; up to 2048 steps (four for each workgroup that is resident) take a few us either way
    const bool fine = (double)at.pairs * (block_size / 64) * p.G <= 2048.0 * 64;
    const void* dkv = fine ? (const void*)&query_attn_dkv_kernel<true> : (const void*)&query_attn_dkv_kernel<false>;
    if (launch(dkv, dim3((unsigned)at.items), kargs, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    return launch((const void*)&query_sum_kernel, dim3(key_tiles), kargs, s) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
