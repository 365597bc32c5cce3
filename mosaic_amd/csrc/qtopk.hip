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
// scores are formed again in fp64, one block per lane, and compared there.
//
// One workgroup = 16 query tokens of one kv head.  Its waves form the scores S^T = K Q^T of up to
// 64 PL blocks with v_mfma_f32_16x16x32_bf16 into LDS (16 rows of fp32), then each wave takes
// rows: PL scores per lane in registers, T by bisection between the row's largest score and the
// smallest of the lanes' largest ones (64 scores at least lie above it, and K <= 64), each step a
// compare and a population count per register, and the indices by their prefix counts.  More
// blocks than 64 PL go in chunks: the rows' best K so far join the next chunk's scores.
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
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ float wave_min(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = fminf(x, __shfl_xor(x, m));
    return x;
}

template <int PL, int NW>
__global__ __launch_bounds__(NW * 64) void query_topk_kernel(QueryTopkParams p) {
    constexpr int kChunk = 64 * PL, kStride = kChunk + 4;
    __shared__ __attribute__((aligned(16))) float sc[kRows * kStride];
    __shared__ float carry_v[kRows][kMaxTopk];   // best K of the chunks so far, ascending blocks
    __shared__ int carry_u[kRows][kMaxTopk];
    __shared__ int carry_n[kRows];
    __shared__ float qnorm[kRows], knorm[NW];
    __shared__ double qd[NW][64];                // a wave's exact summed query (rows that need it)

    const int lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x % p.qtiles, rest = blockIdx.x / p.qtiles;
    const int h = rest % p.Hk, b = rest / p.Hk;
    const int n0 = tile * kRows;
    const bf16_t* kb = p.k + b * p.k_sb + h * p.k_sh;
    const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (int64_t)b * p.nb;

    // the summed query of column c16 (dims 32 ks + 8 g4 .. + 7), as hi + lo operands
    bf16x8 hi[2], lo[2];
    {
        const bf16_t* qb = p.q + b * p.q_sb + (int64_t)min(n0 + c16, p.Nq - 1) * p.q_sn + (int64_t)h * p.G * p.q_sh;
        float sum[2][8], mag = 0.f, tot[2][8];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[ks][i] = tot[ks][i] = 0.f;
        for (int g = 0; g < p.G; ++g)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const uint4 u = ld16(qb + g * p.q_sh + 32 * ks + 8 * g4);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[ks][2 * i] += bf_lo(w[i]);
                    sum[ks][2 * i + 1] += bf_hi(w[i]);
                    tot[ks][2 * i] += fabsf(bf_lo(w[i]));
                    tot[ks][2 * i + 1] += fabsf(bf_hi(w[i]));
                }
            }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = round_bf16(sum[ks][i]);
                hi[ks][i] = (__bf16)a;
                lo[ks][i] = (__bf16)(sum[ks][i] - a);
                mag = fmaf(tot[ks][i], tot[ks][i], mag);
            }
        mag += __shfl_xor(mag, 16);
        mag += __shfl_xor(mag, 32);
        if (wave == 0 && lane < 16) qnorm[lane] = sqrtf(mag);
    }
    const int rows = min(kRows, p.Nq - n0);
    float kn = 0.f;   // largest squared norm of this lane's dims over the blocks it has loaded
    for (int u0 = 0; u0 < p.nb; u0 += kChunk) {
        const int nc = min(kChunk, p.nb - u0);
        for (int t = wave; t < (nc + 15) / 16; t += NW) {
            const int u = u0 + 16 * t + c16;
            const bf16_t* kr = kb + (int64_t)min(u, p.nb - 1) * p.k_sn + 8 * g4;
            const uint4 a0 = ld16(kr), a1 = ld16(kr + 32);
            const bool on = u < p.nb && (mask == nullptr || mask[u]);
            float nn = 0.f;
            const uint32_t aw[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bf16x2 e = __builtin_bit_cast(bf16x2, aw[i]);
                nn = __builtin_amdgcn_fdot2_f32_bf16(e, e, nn, false);
            }
            kn = on ? fmaxf(kn, nn) : kn;
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
            s = mfma16(as_bf16x8(a0), hi[0], s);
            s = mfma16(as_bf16x8(a1), hi[1], s);
            if (p.G > 1) {
                s = mfma16(as_bf16x8(a0), lo[0], s);
                s = mfma16(as_bf16x8(a1), lo[1], s);
            }
            // lane: blocks 16 t + 4 g4 + e of query c16; the flag of block c is lane c's
            const uint32_t ons = (uint32_t)__builtin_amdgcn_ballot_w64(on) >> (4 * g4);
            float4 v;
            v.x = (ons & 1) && s[0] == s[0] ? s[0] : -INFINITY;
            v.y = (ons & 2) && s[1] == s[1] ? s[1] : -INFINITY;
            v.z = (ons & 4) && s[2] == s[2] ? s[2] : -INFINITY;
            v.w = (ons & 8) && s[3] == s[3] ? s[3] : -INFINITY;
            *reinterpret_cast<float4*>(sc + c16 * kStride + 16 * t + 4 * g4) = v;
        }
        {   // |k|^2 <= the sum over the four dim groups of their largest
            float m = kn;
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
            m += __shfl_xor(m, 16);
            m += __shfl_xor(m, 32);
            if (lane == 0) knorm[wave] = m;
        }
        __syncthreads();
        float kmax = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) kmax = fmaxf(kmax, knorm[i]);
        kmax = sqrtf(kmax);
        const bool last = u0 + kChunk >= p.nb;
        for (int r = wave; r < rows; r += NW) {
            // element 0: the carried best, element 1 + i: block u0 + lane + 64 i; -inf past the end
            float v[PL + 1];
            int cu = 0;
            v[0] = -INFINITY;
            if (u0 > 0 && lane < carry_n[r]) {
                v[0] = carry_v[r][lane];
                cu = carry_u[r][lane];
            }
#pragma unroll
            for (int i = 0; i < PL; ++i) v[1 + i] = lane + 64 * i < nc ? sc[r * kStride + lane + 64 * i] : -INFINITY;
            auto count = [&](float x) {   // scores >= x
                int n = 0;
#pragma unroll
                for (int i = 0; i <= PL; ++i) n += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= x));
                return n;
            };
            float top = v[0], low = v[0] == -INFINITY ? INFINITY : v[0];
#pragma unroll
            for (int i = 1; i <= PL; ++i) {
                top = fmaxf(top, v[i]);
                low = fminf(low, v[i] == -INFINITY ? INFINITY : v[i]);
            }
            const float inner = wave_min(top);     // -inf where a lane has no block
            const int valid = count(-__FLT_MAX__);
            float from, to;                        // taken: certainly above `to`, perhaps in [from, to]
            int sure = 0, maybe = valid;
            if (valid <= p.K) {
                from = -__FLT_MAX__;
                to = INFINITY;
            } else {
                float hi_s = wave_max(top), lo_s = inner > -INFINITY ? inner : wave_min(low);
                // count(lo_s) >= K and fewer than K lie above hi_s; T in [lo_s, hi_s]
                float T = hi_s;
                if (count(hi_s) < p.K) {
                    for (;;) {
                        const float mid = 0.5f * lo_s + 0.5f * hi_s;
                        if (!(mid > lo_s && mid < hi_s)) {   // neighbours: ties
                            T = lo_s;
                            break;
                        }
                        const int n = count(mid);
                        if (n == p.K) {
                            float least = INFINITY;
#pragma unroll
                            for (int i = 0; i <= PL; ++i) least = fminf(least, v[i] >= mid ? v[i] : INFINITY);
                            T = wave_min(least);
                            break;
                        }
                        if (n > p.K) lo_s = mid; else hi_s = mid;
                    }
                }
                float e2 = 0x1p-14f * qnorm[r] * kmax;       // 2 eps
                if (!(e2 < INFINITY)) e2 = 0.f;
                from = T - e2;
                to = T + e2;
                maybe = count(from);
#pragma unroll
                for (int i = 0; i <= PL; ++i) sure += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] > to));
                maybe -= sure;
            }
            uint32_t taken = 0;    // bit i: element i
#pragma unroll
            for (int i = 0; i <= PL; ++i) taken |= (v[i] >= from) ? 1u << i : 0u;
            if (sure + maybe > p.K) {
                // exact scores of the blocks between, one per lane at a time
                double* qs = qd[wave];
                {
                    const bf16_t* qb = p.q + b * p.q_sb + (int64_t)(n0 + r) * p.q_sn + (int64_t)h * p.G * p.q_sh + lane;
                    double sum = 0.0;
                    for (int g = 0; g < p.G; ++g) sum += (double)bf2f(qb[g * p.q_sh]);
                    qs[lane] = sum;
                }
                double s[PL + 1];
                uint32_t open = 0;
#pragma unroll
                for (int i = 0; i <= PL; ++i) {
                    s[i] = 0.0;
                    if (v[i] >= from && v[i] <= to) {
                        open |= 1u << i;
                        const bf16_t* kr = kb + (int64_t)(i == 0 ? cu : u0 + lane + 64 * (i - 1)) * p.k_sn;
                        double a = 0.0;
                        for (int d = 0; d < 64; d += 8) {
                            const uint4 w4 = ld16(kr + d);
                            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                a = fma(qs[d + 2 * j], (double)bf_lo(w[j]), a);
                                a = fma(qs[d + 2 * j + 1], (double)bf_hi(w[j]), a);
                            }
                        }
                        s[i] = a;
                    }
                }
                taken &= ~open;
                for (int left = p.K - sure; left > 0; --left) {   // the best of the open ones, the lower block first
                    double best = -INFINITY;
                    int bu = 0x7fffffff, bi = 0;
#pragma unroll
                    for (int i = 0; i <= PL; ++i) {
                        const int u = i == 0 ? cu : u0 + lane + 64 * (i - 1);
                        if ((open >> i & 1) && (s[i] > best || (s[i] == best && u < bu))) {
                            best = s[i];
                            bu = u;
                            bi = i;
                        }
                    }
                    double wb = best;
                    int wu = bu;
#pragma unroll
                    for (int m = 1; m < 64; m <<= 1) {
                        const double ob = __shfl_xor(wb, m);
                        const int ou = __shfl_xor(wu, m);
                        if (ob > wb || (ob == wb && ou < wu)) {
                            wb = ob;
                            wu = ou;
                        }
                    }
                    if (wu == bu && bu != 0x7fffffff) {
                        taken |= 1u << bi;
                        open &= ~(1u << bi);
                    }
                }
            }
            // taken blocks in ascending order: the carried ones, then the chunk's by register and lane
            int at = 0;
            int64_t* row = p.out + (((int64_t)b * p.Nq + n0 + r) * p.Hk + h) * p.K;
#pragma unroll
            for (int i = 0; i <= PL; ++i) {
                const bool on = taken >> i & 1;
                const uint64_t m = __builtin_amdgcn_ballot_w64(on);
                const int pos = at + (int)__builtin_popcountll(m & ((1ull << lane) - 1ull));
                const int u = i == 0 ? cu : u0 + lane + 64 * (i - 1);
                if (on) {
                    if (last) {
                        row[pos] = u;
                    } else {
                        carry_v[r][pos] = v[i];
                        carry_u[r][pos] = u;
                    }
                }
                at += (int)__builtin_popcountll(m);
            }
            if (last) {
                if (lane >= at && lane < p.K) row[lane] = -1;
            } else if (lane == 0) {
                carry_n[r] = at;
            }
        }
        if (!last) __syncthreads();   // the rows' scores are read before the next chunk's are written
    }
}

template <int PL>
const void* topk_fn(bool wide) {
    return wide ? (const void*)&query_topk_kernel<PL, 16> : (const void*)&query_topk_kernel<PL, 4>;
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
    const void* fn = num_blocks <= 256 ? topk_fn<4>(wide) : num_blocks <= 512 ? topk_fn<8>(wide)
                   : num_blocks <= 768 ? topk_fn<12>(wide) : topk_fn<16>(wide);
    void* args[] = {&p};
    return hipLaunchKernel(fn, dim3((unsigned)wgs), dim3(wide ? 1024 : 256), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess
               ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}
