// qcache.hip -- quantising a key/value cache as it is written, and reading it back (gfx950).
//
// A write puts tokens [start, end) of a member into its blocks; its sequence ends there.  For each block
// touched, kv head, and for keys and values on their own, with M the largest code (127, or 448 in e4m3):
//   a     = the largest |x| of the block's new tokens (0 where it is below 2^-100)
//   scale = a / M, and not below the block's scale before where earlier tokens of it are kept
//   code  = x / scale rounded to the nearest code, ties to even; of a kept token, code scale_before / scale
// Tokens of the block behind the end become zeros; other blocks stay as they are.  A value that is not
// finite makes its block's scale NaN, which everything read from the block then is.  The mean of the
// block's keys (the sum of the codes times the scale over the number of tokens) goes to k_mean, where
// query_topk takes it from, and the largest of their norms to k_norm, by which the attention knows where it
// needs no maxima.
//
// The rounding is that of the exact quotient: x * (1 / scale), within 1.5 units of its last place, is taken to
// the nearest number that could be a tie, and moved off it by the sign of the remainder, which an fma gives.
//
// Bound by HBM: a workgroup takes a block of one head, reads its rows once into registers and writes
// both code tiles contiguously, 16 bytes a lane.  The heads of a block are neighbouring workgroups, so
// that the lines of their tokens' rows are read together.  24 members of 49152 tokens and 3 heads in bf16, 906 MB
// in and 453 MB of codes out: 265 to 305 us, 4.5 to 5.1 TB/s, where a copy of 2 GiB reaches 5.0; the vector ALU is as
// busy (23 instructions a value, nine of them the exact quotient, five the means and norms).  One token of each of 24
// members, which reads 64 codes of either kind for it: 4.6 us, most of it the launch and one trip to memory and back.
#include <hip/hip_runtime.h>

#include "qcache.h"

namespace mosaic {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLeast = 0x1p-100f;   // below it a block is zeros: 1 / scale stays in fp32

struct CacheParams {
    mosaic_kv_cache c;
    const void* k; int64_t k_sb, k_sn, k_sh;
    const void* v; int64_t v_sb, v_sn, v_sh;
    void* k_out; void* v_out;      // read: [B, n, Hk, 64]
    const int32_t* starts;         // [B], or null: start
    const int32_t* counts;         // [B], or null: n
    int64_t start;
    int n, units;                  // tokens; blocks (write) or tiles of 64 (read) of a member at most
};

template <typename T> struct Row4;   // four values of a row
template <> struct Row4<bf16_t> {
    static __device__ __forceinline__ float4 load(const bf16_t* p) {
        const uint2 u = ld8(p);
        return make_float4(bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y));
    }
    static __device__ __forceinline__ void store(bf16_t* p, float4 x) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
    }
};
template <> struct Row4<float> {
    static __device__ __forceinline__ float4 load(const float* p) { return *reinterpret_cast<const float4*>(p); }
    static __device__ __forceinline__ void store(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
};

// N values as they lie in memory, and the largest of their magnitudes' bits (NaN above infinity)
template <typename T, int N> struct Raw;
template <int N> struct Raw<bf16_t, N> {
    uint32_t w[N / 2];
    __device__ __forceinline__ void load(const bf16_t* p) {
        if constexpr (N == 4) {
            const uint2 u = ld8(p);
            w[0] = u.x; w[1] = u.y;
        } else
#pragma unroll
            for (int i = 0; i < N / 8; ++i) {
                const uint4 u = ld16(p + 8 * i);
                w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
            }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]); }
    // two magnitudes a word until the end
    __device__ __forceinline__ uint32_t most(uint32_t m) const {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu)));
        return m;
    }
    static __device__ __forceinline__ uint32_t end(uint32_t m) { return max(m & 0xffff0000u, m << 16); }
};
template <int N> struct Raw<float, N> {
    uint32_t w[N];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 u = ld16(p + 4 * i);
            w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(w[i]); }
    __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, w[i] & 0x7fffffffu);
        return m;
    }
    static __device__ __forceinline__ uint32_t end(uint32_t m) { return m; }
};

// y, moved by a few units of its last place towards the side on which the quotient lies: the sign of
// `rest` is that of the quotient minus y, and 0 stays 0.
__device__ __forceinline__ float beside(float y, float rest) {
    return rest == 0.f ? y : fmaf(fabsf(y), copysignf(0x1p-22f, rest), y);
}
// The nearest number to y with four zeros at its end: among such are all the codes and the middles between
// them, and no two lie within the error of x * (1 / scale).
__device__ __forceinline__ float blunt(float y) { return __uint_as_float((__float_as_uint(y) + 8) & ~15u); }

struct Quant {
    float scale, inv;   // inv 0 where the block is zeros or NaN
    __device__ __forceinline__ void init(float s) {
        scale = s;
        inv = s > 0.f ? 1.f / s : 0.f;
    }
    __device__ __forceinline__ float quotient(float x) const {
        const float y = blunt(x * inv);
        return beside(y, fmaf(-y, scale, x));
    }
    // of a code under another scale: code * before is high + low exactly
    __device__ __forceinline__ float requotient(float code, float before) const {
        const float high = code * before, low = fmaf(code, before, -high);
        const float y = blunt(high * inv);
        return beside(y, fmaf(-y, scale, high) + low);
    }
};

template <bool FP8>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
    if constexpr (FP8) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    } else {
        // rounded to a whole number by the sum, whose last byte it then is
        auto round = [](float x) { return __float_as_uint(x + 12582912.f); };
        const uint32_t lo = __builtin_amdgcn_perm(round(b), round(a), 0x0c0c0400), hi = __builtin_amdgcn_perm(round(d), round(c), 0x04000c0c);
        return lo | hi;
    }
}

// Sixteen codes under a block's scale before, set to its scale now
template <bool FP8>
__device__ __forceinline__ void rescale(uint32_t (&w)[4], const Quant& q, float before) {
    if (q.scale == before) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 c = codes_f32<FP8>(w[i]);
        const uint32_t x = pack_codes<FP8>(q.requotient(c.x, before), q.requotient(c.y, before), q.requotient(c.z, before), q.requotient(c.w, before));
        w[i] = q.inv == 0.f ? 0u : x;
    }
}

// words of the four lanes of a quad, transposed: lane i's word j becomes lane j's word i
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4]) {
    const int q = threadIdx.x & 3;
    // exchange with lane ^ 1 the words whose low index bit differs, then with lane ^ 2
    const bool odd = q & 1, high = q & 2;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const uint32_t give = odd ? w[j] : w[j + 1];
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0xb1, 0xf, 0xf, true);   // lane ^ 1
        w[j] = odd ? got : w[j];
        w[j + 1] = odd ? w[j + 1] : got;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t give = high ? w[j] : w[j + 2];
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0x4e, 0xf, 0xf, true);   // lane ^ 2
        w[j] = high ? got : w[j];
        w[j + 2] = high ? w[j + 2] : got;
    }
}

// x of lane ^ D of the same half wave
template <int D>
__device__ __forceinline__ float lane_xor(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_ds_swizzle((int)__float_as_uint(x), D << 10 | 0x1f));
}

// Of 2 N sums a lane keeps the upper or the lower N, with those of lane ^ D added
template <int N, int D>
__device__ __forceinline__ void halve_sums(float (&sum)[16], bool upper) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float keep = upper ? sum[i + N] : sum[i], give = upper ? sum[i] : sum[i + N];
        sum[i] = keep + lane_xor<D>(give);
    }
}

// The scale of a block from the largest magnitude (its bits) of its new tokens
template <bool FP8>
__device__ __forceinline__ float new_scale(uint32_t most, bool keeps, float before) {
    constexpr float kTop = FP8 ? 448.f : 127.f;
    const float a = __uint_as_float(most);
    if (most >= 0x7f800000u || (keeps && !(before < INFINITY))) return NAN;
    const float s = a < kLeast ? 0.f : a / kTop;
    return keeps ? fmaxf(s, before) : s;
}

// What a thread holds of each tile of 64 tokens: of the keys the 16 dims of one token that are its chunk
// of the layout; of the values four dims of four tokens, whose codes four neighbouring lanes then
// exchange, so that each has a chunk.
template <typename T, bool FP8, int SUB>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(CacheParams p) {
    __shared__ uint32_t most[2][kWaves];
    __shared__ float sums[2][64], squares[SUB][kWaves][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % p.c.num_kv_heads, rest = blockIdx.x / p.c.num_kv_heads, unit = rest % p.units, b = rest / p.units;
    constexpr int kBlock = 64 * SUB;
    // the run's place among the positions of the sequence, and what of it lies in the cache
    const int64_t at = p.starts != nullptr ? p.starts[b] : p.start;
    const int count = p.counts != nullptr ? min(max(p.counts[b], 0), p.n) : p.n;
    const int64_t first = at < 0 ? 0 : at, last = at + count < p.c.capacity ? at + count : p.c.capacity;
    const int64_t j64 = first / kBlock + unit;
    if (last <= first || j64 * kBlock >= last) return;
    const int j = (int)j64, t0 = j * kBlock, begin = (int)first - t0, end = (int)(last - t0) < kBlock ? (int)(last - t0) : kBlock;
    // new tokens of the block: [max(begin, 0), end); kept ones: those before
    const bool keeps = begin > 0;
    const int64_t blk = block_at(p.c, b, j, h);
    uint8_t* kc = static_cast<uint8_t*>(p.c.k_codes) + blk * (kBlock * 64);
    uint8_t* vc = static_cast<uint8_t*>(p.c.v_codes) + blk * (kBlock * 64);
    const int kkey = 32 * (wave >> 1) + key_of_row(lane & 31), kdim = 32 * (wave & 1) + 16 * (lane >> 5);
    const int vdim = 4 * (lane >> 2), vkey = 16 * wave + 4 * (lane & 3);
    // chunk of the values' layout that this lane stores: dim vdim + lane % 4, tokens 16 wave ..
    const int vd = vdim + (lane & 3), vchunk = (((wave >> 1) * 2 + (vd >> 5)) * 2 + (wave & 1)) * 32 + (vd & 31);
    const T* kx = static_cast<const T*>(p.k) + b * p.k_sb + h * p.k_sh + kdim;
    const T* vx = static_cast<const T*>(p.v) + b * p.v_sb + h * p.v_sh + vdim;

    Raw<T, 16> k[SUB];
    Raw<T, 4> v[SUB][4];
    uint32_t km = 0, vm = 0;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
        const int tk = 64 * s + kkey;
        if (tk >= begin && tk < end) k[s].load(kx + (t0 + tk - at) * p.k_sn);
        else k[s].clear();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tv = 64 * s + vkey + i;
            if (tv >= begin && tv < end) v[s][i].load(vx + (t0 + tv - at) * p.v_sn);
            else v[s][i].clear();
        }
    }
    // the codes that are kept, as far as they share this lane's chunks
    uint4 kwas[SUB], vwas[SUB];
    const float kold = keeps ? p.c.k_scale[blk] : 0.f, vold = keeps ? p.c.v_scale[blk] : 0.f;
    if (keeps)
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            kwas[s] = reinterpret_cast<const uint4*>(kc + s * kCodeTile)[tid];
            vwas[s] = reinterpret_cast<const uint4*>(vc + s * kCodeTile)[vchunk];
        }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
        km = k[s].most(km);
#pragma unroll
        for (int i = 0; i < 4; ++i) vm = v[s][i].most(vm);
    }
    km = Raw<T, 4>::end(km);
    vm = Raw<T, 4>::end(vm);
    km = wave_max_all_u32(km);
    vm = wave_max_all_u32(vm);
    if (lane == 0) {
        most[0][wave] = km;
        most[1][wave] = vm;
    }
    __syncthreads();   // (what the block held is read by every thread by now)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        km = max(km, most[0][w]);
        vm = max(vm, most[1][w]);
    }
    Quant kq, vq;
    kq.init(new_scale<FP8>(km, keeps, kold));
    vq.init(new_scale<FP8>(vm, keeps, vold));

    // a block of zeros or of NaN: codes of zeros
    if (kq.inv == 0.f)
#pragma unroll
        for (int s = 0; s < SUB; ++s) k[s].clear();
    if (vq.inv == 0.f)
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[s][i].clear();

    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = kq.quotient(k[s][i]);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_codes<FP8>(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
        if (keeps) {
            uint32_t was[4] = {kwas[s].x, kwas[s].y, kwas[s].z, kwas[s].w};
            rescale<FP8>(was, kq, kold);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = 64 * s + kkey < begin ? was[i] : w[i];
        }
        float square = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 c = codes_f32<FP8>(w[i]);
            sum[4 * i] += c.x; sum[4 * i + 1] += c.y; sum[4 * i + 2] += c.z; sum[4 * i + 3] += c.w;
            square = fmaf(c.x, c.x, fmaf(c.y, c.y, fmaf(c.z, c.z, fmaf(c.w, c.w, square))));
        }
        squares[s][wave][lane & 31] = xor32_add(square);   // (both halves the same)
        reinterpret_cast<uint4*>(kc + s * kCodeTile)[tid] = make_uint4(w[0], w[1], w[2], w[3]);

        uint32_t x[4];   // word d: dim vdim + d of this lane's four tokens
#pragma unroll
        for (int d = 0; d < 4; ++d)
            x[d] = pack_codes<FP8>(vq.quotient(v[s][0][d]), vq.quotient(v[s][1][d]), vq.quotient(v[s][2][d]), vq.quotient(v[s][3][d]));
        if (keeps) {
            uint32_t was[4] = {vwas[s].x, vwas[s].y, vwas[s].z, vwas[s].w};
            quad_transpose(was);
            rescale<FP8>(was, vq, vold);
            const int kept = min(max(begin - (64 * s + vkey), 0), 4);   // of the four
            const uint32_t mask = kept == 4 ? ~0u : (1u << (8 * kept)) - 1u;
#pragma unroll
            for (int d = 0; d < 4; ++d) x[d] = (x[d] & ~mask) | (was[d] & mask);
        }
        quad_transpose(x);
        reinterpret_cast<uint4*>(vc + s * kCodeTile)[vchunk] = make_uint4(x[0], x[1], x[2], x[3]);
    }

    // the keys' mean: the sixteen sums over the 32 rows of a half wave, each exchange halving what a lane holds
    halve_sums<8, 16>(sum, lane & 16);
    halve_sums<4, 8>(sum, lane & 8);
    halve_sums<2, 4>(sum, lane & 4);
    halve_sums<1, 2>(sum, lane & 2);
    sum[0] += lane_xor<1>(sum[0]);
    // lane bits 4..1 chose the dim: bit 4 the upper eight of sixteen, and so on
    const int dim = kdim + 8 * ((lane >> 4) & 1) + 4 * ((lane >> 3) & 1) + 2 * ((lane >> 2) & 1) + ((lane >> 1) & 1);
    if ((lane & 1) == 0) sums[wave >> 1][dim] = sum[0];
    __syncthreads();
    if (tid < 32) {
        // (the mean of the codes first: their sum times the scale need not fit)
        const float a = (sums[0][2 * tid] + sums[1][2 * tid]) / (float)end * kq.scale;
        const float c = (sums[0][2 * tid + 1] + sums[1][2 * tid + 1]) / (float)end * kq.scale;
        static_cast<uint32_t*>(p.c.k_mean)[blk * 32 + tid] = pack_bf16x2(a, c);
    }
    if (wave == 1) {   // the largest norm of a key: waves 0 and 1, 2 and 3 have the halves of a token
        float square = 0.f;
#pragma unroll
        for (int s = 0; s < SUB; ++s) square = fmaxf(square, squares[s][2 * (lane >> 5)][lane & 31] + squares[s][2 * (lane >> 5) + 1][lane & 31]);
        square = wave_max_nonneg(square);
        if (lane == 0) p.c.k_norm[blk] = sqrtf(square) * kq.scale;
    }
    if (tid == 0) {
        p.c.k_scale[blk] = kq.scale;
        p.c.v_scale[blk] = vq.scale;
    }
}

// The write's exchange backwards; a workgroup takes a tile of 64 tokens of one head.  Tokens outside
// the cache are zeros.  Bound by HBM: 24 members of 49152 tokens and 3 heads to bf16, 453 MB of codes in, half of them
// still in the last cache after a write, and 906 MB out: 220 us; 196608 tokens to fp32, 75 MB in and 302 MB out: 66 us,
// 5.7 TB/s.  (Stores that pass the caches by take half as long again.)
template <typename T, bool FP8>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(CacheParams p) {
    __shared__ uint4 keys[64][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % p.c.num_kv_heads, rest = blockIdx.x / p.c.num_kv_heads, unit = rest % p.units, b = rest / p.units;
    const int64_t at = p.starts != nullptr ? p.starts[b] : p.start;
    const int64_t t0 = ((at >> 6) + unit) * 64;    // (>> rounds down, also before the first token)
    if (t0 >= at + p.n) return;
    const bool held = t0 >= 0 && t0 < (int64_t)p.c.num_blocks * p.c.block_size;
    float ks = 0.f, vs = 0.f;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    const int vdim = 4 * (lane >> 2), vkey = 16 * wave + 4 * (lane & 3);
    if (held) {
        const int j = (int)(t0 / p.c.block_size), sub = ((int)t0 - j * p.c.block_size) / 64;
        const int64_t blk = block_at(p.c, b, j, h), from = blk * p.c.block_size * 64 + sub * kCodeTile;
        const int vd = vdim + (lane & 3), vchunk = (((wave >> 1) * 2 + (vd >> 5)) * 2 + (wave & 1)) * 32 + (vd & 31);
        k = ld16(static_cast<const uint8_t*>(p.c.k_codes) + from + 16 * tid);
        v = ld16(static_cast<const uint8_t*>(p.c.v_codes) + from + 16 * vchunk);
        ks = p.c.k_scale[blk];
        vs = p.c.v_scale[blk];
    }
    const int64_t end = at + p.n < p.c.capacity ? at + p.n : p.c.capacity;
    auto row = [&](void* out, int64_t t, int dim) {
        return static_cast<T*>(out) + (((int64_t)b * p.n + (t - at)) * p.c.num_kv_heads + h) * 64 + dim;
    };
    auto times = [](float4 c, float s) { return make_float4(c.x * s, c.y * s, c.z * s, c.w * s); };
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    // keys: by way of LDS, so that a wave stores whole rows (64 bytes a token, its 16-byte chunks moved by token)
    const int key = 32 * (wave >> 1) + key_of_row(lane & 31);
    keys[key][(2 * (wave & 1) + (lane >> 5)) ^ (key >> 1 & 3)] = k;
    __syncthreads();
    constexpr int kDims = 16 / sizeof(T), kLanes = 64 / kDims;   // of one store, lanes of a row
#pragma unroll
    for (int i = 0; i < 64 * kLanes / kThreads; ++i) {
        const int token = tid / kLanes + i * (kThreads / kLanes), d = tid % kLanes * kDims;
        const int64_t t = t0 + token;
        if (t < at || t >= at + p.n) continue;
        const uint8_t* from = reinterpret_cast<const uint8_t*>(&keys[token][(d >> 4) ^ (token >> 1 & 3)]) + (d & 15);
        const bool in = t >= 0 && t < end;
        T* out = row(p.k_out, t, d);
        if constexpr (sizeof(T) == 2) {
            const uint2 u = ld8(from);
            const float4 x = in ? times(codes_f32<FP8>(u.x), ks) : zero, y = in ? times(codes_f32<FP8>(u.y), ks) : zero;
            *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
        } else Row4<T>::store(out, in ? times(codes_f32<FP8>(*reinterpret_cast<const uint32_t*>(from)), ks) : zero);
    }
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    quad_transpose(w);   // word d: dim vdim + d of tokens vkey ..
    float4 x[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) x[d] = times(codes_f32<FP8>(w[d]), vs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + vkey + i;
        if (t < at || t >= at + p.n) continue;
        auto pick = [&](const float4& y) { return i == 0 ? y.x : i == 1 ? y.y : i == 2 ? y.z : y.w; };
        const bool in = t >= 0 && t < end;
        Row4<T>::store(row(p.v_out, t, vdim), in ? make_float4(pick(x[0]), pick(x[1]), pick(x[2]), pick(x[3])) : zero);
    }
}

// ------------------------------------------------------------------ host

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_rows(const mosaic_bnhd& t, int dtype) {
    const int64_t unit = dtype == MOSAIC_DTYPE_BF16 ? 8 : 4;
    if (t.ptr == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!aligned(t.ptr, 16) || t.stride_b % unit || t.stride_n % unit || t.stride_h % unit) return MOSAIC_ERR_ALIGNMENT;
    return MOSAIC_OK;
}

// Units of `size` tokens that a run of n touches at most
int64_t units_of(int64_t n, int64_t size, int64_t start, bool anywhere) {
    if (anywhere) return (n + size - 2) / size + 1;
    return (start + n + size - 1) / size - start / size;
}

template <typename T, bool FP8>
const void* write_kernel(int bs) {
    return bs == 64    ? (const void*)&kv_cache_write_kernel<T, FP8, 1>
           : bs == 128 ? (const void*)&kv_cache_write_kernel<T, FP8, 2>
                       : (const void*)&kv_cache_write_kernel<T, FP8, 4>;
}

int check_run(const mosaic_kv_cache* cache, int32_t dtype, int32_t head_dim, int32_t n, int64_t start, const int32_t* starts,
              const int32_t* counts) {
    if (int e = check_cache(cache)) return e;
    if (head_dim != kHeadDim) return MOSAIC_ERR_HEAD_DIM;
    if (dtype != MOSAIC_DTYPE_BF16 && dtype != MOSAIC_DTYPE_F32) return MOSAIC_ERR_UNSUPPORTED;
    if (n <= 0) return MOSAIC_ERR_SHAPE;
    if (starts == nullptr && (start < 0 || start > (int64_t)cache->capacity - n)) return MOSAIC_ERR_SHAPE;
    if (!aligned(starts, 4) || !aligned(counts, 4)) return MOSAIC_ERR_ALIGNMENT;
    return MOSAIC_OK;
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

int mosaic_kv_cache_write(const mosaic_kv_cache* cache, mosaic_bnhd k, mosaic_bnhd v, int32_t dtype, int32_t head_dim,
                          int32_t num_tokens, int64_t start, const int32_t* starts, const int32_t* counts, void* stream) {
    if (int e = check_run(cache, dtype, head_dim, num_tokens, start, starts, counts)) return e;
    for (const mosaic_bnhd* t : {&k, &v})
        if (int e = check_rows(*t, dtype)) return e;
    CacheParams p{};
    p.c = *cache;
    p.k = k.ptr; p.k_sb = k.stride_b; p.k_sn = k.stride_n; p.k_sh = k.stride_h;
    p.v = v.ptr; p.v_sb = v.stride_b; p.v_sn = v.stride_n; p.v_sh = v.stride_h;
    p.starts = starts; p.counts = counts; p.start = start; p.n = num_tokens;
    int64_t units = units_of(num_tokens, cache->block_size, start, starts != nullptr);
    if (units > cache->num_blocks) units = cache->num_blocks;
    if (!grid_fits(units * cache->num_kv_heads * cache->batch, kThreads)) return MOSAIC_ERR_SHAPE;
    p.units = (int)units;
    const bool fp8 = cache->code_type == MOSAIC_CODE_E4M3, half = dtype == MOSAIC_DTYPE_BF16;
    const void* fn = half ? (fp8 ? write_kernel<bf16_t, true>(cache->block_size) : write_kernel<bf16_t, false>(cache->block_size))
                          : (fp8 ? write_kernel<float, true>(cache->block_size) : write_kernel<float, false>(cache->block_size));
    void* args[] = {&p};
    const unsigned grid = (unsigned)(units * cache->num_kv_heads * cache->batch);
    return hipLaunchKernel(fn, dim3(grid), dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

int mosaic_kv_cache_read(const mosaic_kv_cache* cache, int32_t dtype, int32_t head_dim, int32_t num_tokens, int64_t start,
                         const int32_t* starts, void* k_out, void* v_out, void* stream) {
    if (int e = check_run(cache, dtype, head_dim, num_tokens, start, starts, nullptr)) return e;
    if (k_out == nullptr || v_out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return MOSAIC_ERR_ALIGNMENT;
    CacheParams p{};
    p.c = *cache;
    p.k_out = k_out; p.v_out = v_out;
    p.starts = starts; p.start = start; p.n = num_tokens;
    const int64_t units = units_of(num_tokens, 64, start, starts != nullptr);
    if ((double)units * cache->num_kv_heads * cache->batch > 2147483647.0 || !grid_fits(units * cache->num_kv_heads * cache->batch, kThreads)) return MOSAIC_ERR_SHAPE;
    p.units = (int)units;
    const bool fp8 = cache->code_type == MOSAIC_CODE_E4M3, half = dtype == MOSAIC_DTYPE_BF16;
    const void* fn = half ? (fp8 ? (const void*)&kv_cache_read_kernel<bf16_t, true> : (const void*)&kv_cache_read_kernel<bf16_t, false>)
                          : (fp8 ? (const void*)&kv_cache_read_kernel<float, true> : (const void*)&kv_cache_read_kernel<float, false>);
    void* args[] = {&p};
    const unsigned grid = (unsigned)(units * cache->num_kv_heads * cache->batch);
    return hipLaunchKernel(fn, dim3(grid), dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
