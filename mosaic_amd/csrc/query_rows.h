// query_rows.h -- what the attentions of query tokens share: the rows of a wave, the order in which tokens
// with key blocks of their own are taken, and the union of the blocks of a workgroup's tokens.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "bsa_common.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32;          // rows (token, head) of a wave
constexpr int kUnion = 1024;       // blocks whose members are marked at a time
constexpr int kMaxSplit = 32;
constexpr int kBuckets = 4096;     // of the order of tokens
constexpr float kTau = 8.f;        // a row's reference moves when a score exceeds it by 2^kTau

// Query tokens, and the key blocks of each
struct QuerySets {
    const int64_t* idx;        // [B, Nq, Hk, K]
    const int32_t* lens;       // [B] keys of each sequence, or null
    uint16_t* keys;            // [B, Hk, Nq] bucket of each token (null: tokens in their own order)
    int32_t* order;            // [B, Hk, Nq] tokens in the order they are taken in,
    int32_t* ordered;          // [B, Hk] where this is not 0
    int B, Nq, Nk, Hq, Hk, G, QW, bs, K, nb;
    int qtiles, splits;
    int qw_inverse;            // t / QW = t qw_inverse >> 16 for t < 256
};

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

__device__ __forceinline__ int seq_keys(const QuerySets& p, int b) {
    return p.lens == nullptr ? p.Nk : min(max(p.lens[b], 0), p.Nk);
}

// ------------------------------------------------------------------ the order of tokens
// Tokens of one kv head by a block of theirs: the one nearest the mean of them, in whatever order
// the row has them.  (10007 stations whose rows are in the order of scores: 22.0 blocks in a
// workgroup's union, as by the median; by the row's middle entry 31.7, by the mean itself 24.1.)

__device__ __forceinline__ int bucket_of(const QuerySets& p, int blk) {
    return p.nb <= kBuckets ? blk : (int)((int64_t)blk * kBuckets / p.nb);
}

// Where the tokens' own order is already one of neighbours it is left as it is.  It is one if, of up to 64
// pairs of tokens that follow one another and have entries, at most a quarter have middle entries further apart than a 32nd
// of the blocks.  Every workgroup looks at the same pairs, then takes 32 tokens of one (b, h), eight lanes a
// token.  (49152 tokens that stay: 6 us, and 10 where each is read for it.)
constexpr int kKeyTokens = kThreads / 8;
__global__ __launch_bounds__(kThreads) void query_keys_kernel(QuerySets p, int chunks) {
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
__global__ __launch_bounds__(kOrderThreads) void query_order_kernel(QuerySets p) {
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

// ------------------------------------------------------------------ the union of a workgroup's sets

struct UnionLds {
    __attribute__((aligned(16))) uint32_t members[kUnion][kWaves];   // bit t: token t of the wave has the block
    uint16_t list[kUnion];
    int tokens[kWaves * kRows];
    int found[kWaves];
};

// The workgroup's tokens (positions n0 .. of the order) into LDS; ends with a barrier.
__device__ __forceinline__ void load_tokens(const QuerySets& p, UnionLds& L, int b, int h, int n0) {
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
__device__ __forceinline__ int unite(const QuerySets& p, UnionLds& L, int b, int h, int n0, int end, int c0, int nc,
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

// ------------------------------------------------------------------ rows

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
    __device__ __forceinline__ void init(const QuerySets& p, const Tokens& tokens, int b, int h, int n0, int wave, int r) {
        token = r / p.G;
        live = token < p.QW && n0 + wave * p.QW + token < p.Nq;
        head = h * p.G + (live ? r - token * p.G : 0);
        n = tokens(wave * p.QW + (live ? token : 0));
        at = ((int64_t)b * p.Nq + n) * p.Hq + head;
    }
    __device__ __forceinline__ bool in(uint32_t members) const { return live && (members >> token & 1); }
};

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

// Whether every element of x is finite (their difference with themselves is 0)
__device__ __forceinline__ bool finite(const f32x16& x) {
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) d = fmaf(0.f, x[e], d);
    return d == 0.f;
}

// ------------------------------------------------------------------ host

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

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

// Whether tokens may be taken in another order: with more than one workgroup of them.
bool may_order(int32_t nq, int32_t hq, int32_t hk) { return nq > kWaves * (kRows / (hq / hk)); }
int key_chunks(int32_t nq) { return (nq + kKeyTokens - 1) / kKeyTokens; }
size_t order_bytes(int32_t batch, int32_t nq, int32_t hq, int32_t hk) {
    if (!may_order(nq, hq, hk)) return 0;
    const size_t rows = (size_t)batch * hk * nq;
    return up(rows * sizeof(uint16_t)) + up(rows * sizeof(int32_t)) + up((size_t)batch * hk * sizeof(int32_t));
}
void place_order(QuerySets& p, char* ws) {
    if (!may_order(p.Nq, p.Hq, p.Hk)) return;
    const size_t rows = (size_t)p.B * p.Hk * p.Nq;
    p.keys = reinterpret_cast<uint16_t*>(ws);
    p.order = reinterpret_cast<int32_t*>(ws + up(rows * sizeof(uint16_t)));
    p.ordered = reinterpret_cast<int32_t*>(ws + up(rows * sizeof(uint16_t)) + up(rows * sizeof(int32_t)));
}

hipError_t launch(const void* fn, dim3 grid, void** args, hipStream_t s, int threads = kThreads) {
    return hipLaunchKernel(fn, grid, dim3(threads), args, 0, s);
}

int launch_order(QuerySets& p, hipStream_t s) {
    if (p.keys == nullptr) return MOSAIC_OK;
    int chunks = key_chunks(p.Nq);
    void* args[] = {&p, &chunks};
    if (launch((const void*)&query_keys_kernel, dim3(p.B * p.Hk * chunks), args, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    return launch((const void*)&query_order_kernel, dim3(p.B * p.Hk), args, s, kOrderThreads) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // namespace
}  // namespace mosaic
