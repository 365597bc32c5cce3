// rotary.hip -- rotary positions with several axes, and the RMS norm of each query and key head
// with its rotation, forward and backward, as one pass over q and k (gfx950).
//
// A head x of D dimensions holds D/2 pairs: (2i, 2i+1) interleaved, or (i, i + D/2) as halves.
// Pair i belongs to an axis of the position; with the axis's n pairs numbered j = 0 .. n-1 its
// angle is  a_i = position[axis] * theta_axis^(-j/n).  Pairs past the last axis stay as they are.
//   rotation   y = R(a) x:  y0 = x0 cos a - x1 sin a,  y1 = x1 cos a + x0 sin a
//   with norm  y = R(a) (w h),  h = x r,  r = rsqrt(mean(x^2) + eps)
//   backward   u = R(-a) g;  without norm dx = u;  with it
//              dw = sum over tokens and heads of u h,   v = w u,   dx = r (v - h mean(v h))
// Statistics and sums are fp32, every output is rounded once to its type.
//
// Angles come from the caller's cos / sin tables ([N, D/2] fp32, as the RoPE module keeps them)
// or from the positions.  A far position loses its angle in fp32 (position 10^6 at frequency 1 is
// known to 0.06 radians), so the position times the pair's frequency in turns is an fp64 product,
// its whole turns are taken off in fp64, and only the rest of half a turn at most goes to the
// fp32 sine and cosine (absolute error about 2e-7).
//
// Bound by HBM: q and k are read once and written once (the norm's backward reads x and g).  A
// group of D/8 lanes owns one token: a lane holds the same 8 dimensions of every head, so its
// cosines and sines are formed once and used by all heads, and the norm is a sum over the group.
// Four heads' loads are in flight per lane.  196608 tokens of 12 + 3 heads of 64 in bf16 (757 MB) take
// 149 us, 5.1 TB/s, and as many with the norm (sequence-first) 151, where a copy of 1 GiB reaches
// 5.2; the norm's backward on 49152 tokens of 16 + 4 heads (378 MB) 72 us and 5 for the weights'.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "bsa_common.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kThreads = 256;
constexpr int kHeadRun = 4;        // heads whose loads are in flight together
constexpr int kMaxPairs = 64;      // D <= 128
constexpr int kMaxBwdGroups = 2048;  // workgroups (rows of weight-gradient partials) of the norm's backward

struct RotTensor {
    const void* x; int64_t sb, sn, sh;   // forward input (the norm's backward: x)
    const void* g; int64_t gsb, gsn, gsh;  // gradient of the output (the norm's backward)
    void* y;                             // [B, N, H, D] contiguous
    const float* w;                      // [D] or null
    int heads;
};

struct RotParams {
    RotTensor t[2];                      // q, k
    int N, tokens;                       // tokens = B * N
    int splits, chunks;                  // items per token, runs of kHeadRun heads (q's, then k's)
    float eps, sign;                     // sign -1 turns back
    const float* cos_t; const float* sin_t;              // tables, or null
    const void* pos; int pos_type; int64_t pos_sb, pos_sn;   // positions, or null
    int pairs;                           // rotated pairs
    double turns[kMaxPairs];             // frequency of each pair / (2 pi)
    int8_t axis[kMaxPairs];
    float* partial;                      // [workgroups, 2, D] weight-gradient partials, or null
};

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16_t* p, float (&v)[8]) {
    const uint4 u = ld16(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(w[i]); v[2 * i + 1] = bf_hi(w[i]); }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// sum over each group of GL consecutive lanes (4, 8 or 16), in every lane of it
template <int GL>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
    for (int m = 1; m < GL; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

__device__ __forceinline__ double position(const RotParams& p, int64_t at) {
    switch (p.pos_type) {
        case MOSAIC_POS_F32: return (double)static_cast<const float*>(p.pos)[at];
        case MOSAIC_POS_F64: return static_cast<const double*>(p.pos)[at];
        case MOSAIC_POS_I32: return (double)static_cast<const int32_t*>(p.pos)[at];
        default: return (double)static_cast<const int64_t*>(p.pos)[at];
    }
}

// Cosines and sines of a lane's pairs: interleaved, the 4 pairs of its 8 dimensions; halves, the
// 8 pairs its dimensions take part in (both halves' lanes hold the same ones).
template <int D, bool INTER>
struct Turn {
    static constexpr int NP = INTER ? 4 : 8;
    float c[NP], s[NP];
    int first;   // first pair of this lane

    __device__ __forceinline__ void set(const RotParams& p, int b, int n, int lg) {
        first = INTER ? 4 * lg : 8 * (lg & (D / 16 - 1));
        if (p.cos_t != nullptr) {
#pragma unroll
            for (int i = 0; i < NP; i += 4) {
                const int64_t at = (int64_t)n * (D / 2) + first + i;
                const float4 cv = *reinterpret_cast<const float4*>(p.cos_t + at);
                const float4 sv = *reinterpret_cast<const float4*>(p.sin_t + at);
                c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
                s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int pair = first + i;
                c[i] = 1.f;
                s[i] = 0.f;
                if (pair < p.pairs) {
                    const double t = position(p, b * p.pos_sb + n * p.pos_sn + p.axis[pair]) * p.turns[pair];
                    sincospif(2.f * (float)(t - rint(t)), &s[i], &c[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) s[i] *= p.sign;
    }

    // v turned in place; pairs past the rotated ones are kept as they are, whatever their partner
    __device__ __forceinline__ void apply(float (&v)[8], int pairs, int lg) const {
        if constexpr (INTER) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = v[2 * i], b = v[2 * i + 1];
                const bool on = first + i < pairs;
                v[2 * i] = on ? rope_mul_sub(a, c[i], b, s[i]) : a;
                v[2 * i + 1] = on ? rope_mul_add(b, c[i], a, s[i]) : b;
            }
        } else {
            const bool upper = lg >= D / 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = v[i], b = __shfl_xor(a, D / 16);
                const float y = upper ? rope_mul_add(a, c[i], b, s[i]) : rope_mul_sub(a, c[i], b, s[i]);
                v[i] = first + i < pairs ? y : a;
            }
        }
    }
};

// The runs of heads of one item: run r of p.chunks covers heads [h0, h0 + count) of tensor ti.
__device__ __forceinline__ void head_run(const RotParams& p, int r, int& ti, int& h0, int& count) {
    const int qr = (p.t[0].heads + kHeadRun - 1) / kHeadRun;
    ti = r >= qr ? 1 : 0;
    h0 = (ti ? r - qr : r) * kHeadRun;
    count = min(kHeadRun, p.t[ti].heads - h0);
}

template <typename T, int D, bool INTER, bool NORM>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotParams p) {
    constexpr int GL = D / 8;
    const int lg = threadIdx.x % GL;
    const int64_t items = (int64_t)p.tokens * p.splits;
    float w[2][8];
    if constexpr (NORM) {
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[ti][i] = p.t[ti].w != nullptr ? p.t[ti].w[8 * lg + i] : 1.f;
    }
    const int64_t step = (int64_t)gridDim.x * (kThreads / GL);
    for (int64_t item = (int64_t)blockIdx.x * (kThreads / GL) + threadIdx.x / GL; item < items; item += step) {
        const int tok = (int)(item / p.splits), part = (int)(item - (int64_t)tok * p.splits);
        const int b = tok / p.N, n = tok - b * p.N;
        const int r1 = p.splits == 1 ? p.chunks : part + 1;
        Turn<D, INTER> turn;
        bool turned = false;
        for (int r = part; r < r1; ++r) {
            int ti, h0, count;
            head_run(p, r, ti, h0, count);
            const T* x = static_cast<const T*>(ti ? p.t[1].x : p.t[0].x) + b * (ti ? p.t[1].sb : p.t[0].sb) +
                         n * (ti ? p.t[1].sn : p.t[0].sn) + 8 * lg;
            const int64_t sh = ti ? p.t[1].sh : p.t[0].sh;
            T* y = static_cast<T*>(ti ? p.t[1].y : p.t[0].y) +
                   ((int64_t)tok * (ti ? p.t[1].heads : p.t[0].heads) + h0) * D + 8 * lg;
            float v[kHeadRun][8];
#pragma unroll
            for (int h = 0; h < kHeadRun; ++h)   // past the last head: the last one again, not stored
                load8(x + (h0 + min(h, count - 1)) * sh, v[h]);
            if (!turned) {
                turn.set(p, b, n, lg);
                turned = true;
            }
#pragma unroll
            for (int h = 0; h < kHeadRun; ++h) {
                if constexpr (NORM) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(v[h][i], v[h][i], ss);
                    const float rs = 1.f / sqrtf(group_sum<GL>(ss) * (1.f / D) + p.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[h][i] = v[h][i] * rs * (ti ? w[1][i] : w[0][i]);
                }
                turn.apply(v[h], p.pairs, lg);
                if (h < count) store8(y + h * D, v[h]);
            }
        }
    }
}

// Backward with the norm.  A lane's weight gradients (its 8 dimensions, q's and k's) stay in
// registers over all of its tokens; the workgroup adds its groups in LDS in a fixed order and
// writes one row of partials, and wgrad_kernel adds the rows: no atomics, so the result does not
// depend on the order in which workgroups run.
template <typename T, int D, bool INTER>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(RotParams p) {
    constexpr int GL = D / 8, GROUPS = kThreads / GL;
    __shared__ float part_w[GROUPS][2 * D];
    const int lg = threadIdx.x % GL;
    float w[2][8], dw[2][8];
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[ti][i] = p.t[ti].w != nullptr ? p.t[ti].w[8 * lg + i] : 1.f;
            dw[ti][i] = 0.f;
        }
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    for (int64_t tok64 = (int64_t)blockIdx.x * GROUPS + threadIdx.x / GL; tok64 < p.tokens; tok64 += step) {
        const int tok = (int)tok64;
        const int b = tok / p.N, n = tok - b * p.N;
        Turn<D, INTER> turn;
        turn.set(p, b, n, lg);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const RotTensor& t = p.t[ti];
            const T* x = static_cast<const T*>(t.x) + b * t.sb + n * t.sn + 8 * lg;
            const T* g = static_cast<const T*>(t.g) + b * t.gsb + n * t.gsn + 8 * lg;
            T* y = static_cast<T*>(t.y) + (int64_t)tok * t.heads * D + 8 * lg;
            for (int h0 = 0; h0 < t.heads; h0 += 2) {
                float xv[2][8], gv[2][8];
                const int h1 = min(h0 + 1, t.heads - 1);
                load8(x + h0 * t.sh, xv[0]);
                load8(g + h0 * t.gsh, gv[0]);
                load8(x + h1 * t.sh, xv[1]);
                load8(g + h1 * t.gsh, gv[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(xv[h][i], xv[h][i], ss);
                    const float rs = 1.f / sqrtf(group_sum<GL>(ss) * (1.f / D) + p.eps);
                    turn.apply(gv[h], p.pairs, lg);
                    float m = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        xv[h][i] *= rs;                                  // h
                        m = fmaf(gv[h][i] * w[ti][i], xv[h][i], m);      // v h
                    }
                    m = group_sum<GL>(m) * (1.f / D);
                    if (h0 + h < t.heads) {
                        float dx[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            dw[ti][i] = fmaf(gv[h][i], xv[h][i], dw[ti][i]);
                            dx[i] = rs * (gv[h][i] * w[ti][i] - xv[h][i] * m);
                        }
                        store8(y + (h0 + h) * D, dx);
                    }
                }
            }
        }
    }
    if (p.partial == nullptr) return;
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int i = 0; i < 8; ++i) part_w[threadIdx.x / GL][ti * D + 8 * lg + i] = dw[ti][i];
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += kThreads) {
        float s = 0.f;
        for (int g = 0; g < GROUPS; ++g) s += part_w[g][c];
        p.partial[(int64_t)blockIdx.x * 2 * D + c] = s;
    }
}

// Column sums of the partials [rows, 2 D] -> q's [D] and k's [D] (either may be null): a workgroup
// takes 8 columns, 32 rows at a time, eight loads a thread in flight (2048 rows: 5.5 us; one at a time 10.8).
__global__ __launch_bounds__(kThreads) void wgrad_kernel(const float* partial, int rows, int D, float* dwq, float* dwk) {
    __shared__ float part[32][9];
    const int c = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    const int col = 8 * blockIdx.x + c;
    float s[8] = {};   // eight loads in flight
    for (int r = r0; r < rows; r += 256)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = r + 32 * i;
            const float x = partial[(int64_t)min(at, rows - 1) * 2 * D + col];
            s[i] += at < rows ? x : 0.f;
        }
    part[r0][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (r0 == 0) {
        float sum = 0.f;
        for (int r = 0; r < 32; ++r) sum += part[r][c];
        float* out = col < D ? dwq : dwk;
        if (out != nullptr) out[col < D ? col : col - D] = sum;
    }
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_rows(const mosaic_bnhd& t, int dtype) {
    if (t.ptr == nullptr) return MOSAIC_ERR_NULL_POINTER;
    const int unit = dtype == MOSAIC_DTYPE_F32 ? 4 : 8;
    if (!aligned(t.ptr, 16) || t.stride_b % unit || t.stride_n % unit || t.stride_h % unit) return MOSAIC_ERR_ALIGNMENT;
    return MOSAIC_OK;
}

int fill_rotation(RotParams& p, const mosaic_rotation* rot, int D) {
    p.sign = 1.f;
    if (rot == nullptr) return MOSAIC_OK;
    if (rot->cos != nullptr || rot->sin != nullptr) {
        if (rot->cos == nullptr || rot->sin == nullptr) return MOSAIC_ERR_NULL_POINTER;
        if (!aligned(rot->cos, 16) || !aligned(rot->sin, 16)) return MOSAIC_ERR_ALIGNMENT;
        p.cos_t = rot->cos;
        p.sin_t = rot->sin;
        p.pairs = D / 2;
        return MOSAIC_OK;
    }
    if (rot->positions == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (rot->num_axes < 1 || rot->num_axes > MOSAIC_MAX_AXES) return MOSAIC_ERR_SHAPE;
    if (rot->position_type < MOSAIC_POS_F32 || rot->position_type > MOSAIC_POS_I64) return MOSAIC_ERR_MODE;
    const int size = rot->position_type == MOSAIC_POS_F32 || rot->position_type == MOSAIC_POS_I32 ? 4 : 8;
    if (!aligned(rot->positions, size)) return MOSAIC_ERR_ALIGNMENT;
    p.pos = rot->positions;
    p.pos_type = rot->position_type;
    p.pos_sb = rot->stride_b;
    p.pos_sn = rot->stride_n;
    const double two_pi = 6.283185307179586476925286766559;
    for (int a = 0; a < rot->num_axes; ++a) {
        const int n = rot->sections[a];
        if (n < 0 || p.pairs + n > D / 2) return MOSAIC_ERR_SHAPE;
        if (!(rot->theta[a] > 0.0) || !std::isfinite(rot->theta[a])) return MOSAIC_ERR_SHAPE;
        for (int j = 0; j < n; ++j, ++p.pairs) {
            p.turns[p.pairs] = std::pow(rot->theta[a], -(double)j / n) / two_pi;
            p.axis[p.pairs] = (int8_t)a;
        }
    }
    return MOSAIC_OK;
}

int check_shape(int32_t dtype, int32_t batch, int32_t seq_len, int32_t hq, int32_t hk, int32_t D) {
    if (dtype != MOSAIC_DTYPE_F32 && dtype != MOSAIC_DTYPE_BF16) return MOSAIC_ERR_MODE;
    if (batch <= 0 || seq_len <= 0 || (int64_t)batch * seq_len > 0x7fffffff) return MOSAIC_ERR_SHAPE;
    if (hq <= 0 || hk < 0 || hq > 65535 || hk > 65535) return MOSAIC_ERR_HEADS;
    if (D != 32 && D != 64 && D != 128) return MOSAIC_ERR_UNSUPPORTED;
    return MOSAIC_OK;
}

template <typename T, int D>
const void* rotate_fn(bool inter, bool norm) {
    if (inter) return norm ? (const void*)&rotate_kernel<T, D, true, true> : (const void*)&rotate_kernel<T, D, true, false>;
    return norm ? (const void*)&rotate_kernel<T, D, false, true> : (const void*)&rotate_kernel<T, D, false, false>;
}
template <typename T, int D>
const void* bwd_fn(bool inter) {
    return inter ? (const void*)&norm_bwd_kernel<T, D, true> : (const void*)&norm_bwd_kernel<T, D, false>;
}
template <typename T>
const void* pick(int D, bool inter, bool norm, bool bwd) {
    if (bwd) return D == 32 ? bwd_fn<T, 32>(inter) : D == 64 ? bwd_fn<T, 64>(inter) : bwd_fn<T, 128>(inter);
    return D == 32 ? rotate_fn<T, 32>(inter, norm) : D == 64 ? rotate_fn<T, 64>(inter, norm) : rotate_fn<T, 128>(inter, norm);
}

int bwd_groups(int64_t tokens, int D) {
    const int64_t per = kThreads / (D / 8);
    const int64_t n = (tokens + per - 1) / per;
    return (int)(n < kMaxBwdGroups ? n : kMaxBwdGroups);
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" {

int mosaic_qk_rotate_fwd(mosaic_bnhd q, mosaic_bnhd k, int32_t dtype, int32_t batch, int32_t seq_len,
                         int32_t num_q_heads, int32_t num_k_heads, int32_t head_dim, const mosaic_rotation* rotation,
                         int32_t backward, int32_t norm, const float* q_weight, const float* k_weight, float eps,
                         void* q_out, void* k_out, void* stream) {
    if (int e = check_shape(dtype, batch, seq_len, num_q_heads, num_k_heads, head_dim)) return e;
    if (norm && (backward || !(eps >= 0.f))) return MOSAIC_ERR_MODE;
    if (rotation == nullptr && !norm) return MOSAIC_ERR_NULL_POINTER;
    if (int e = check_rows(q, dtype)) return e;
    if (q_out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (num_k_heads > 0) {
        if (int e = check_rows(k, dtype)) return e;
        if (k_out == nullptr) return MOSAIC_ERR_NULL_POINTER;
    }
    if (!aligned(q_out, 16) || !aligned(k_out, 16) || !aligned(q_weight, 4) || !aligned(k_weight, 4)) return MOSAIC_ERR_ALIGNMENT;
    RotParams p{};
    if (int e = fill_rotation(p, rotation, head_dim)) return e;
    if (backward) p.sign = -1.f;
    p.t[0].x = q.ptr; p.t[0].sb = q.stride_b; p.t[0].sn = q.stride_n; p.t[0].sh = q.stride_h;
    p.t[0].y = q_out; p.t[0].w = q_weight; p.t[0].heads = num_q_heads;
    p.t[1].x = k.ptr; p.t[1].sb = k.stride_b; p.t[1].sn = k.stride_n; p.t[1].sh = k.stride_h;
    p.t[1].y = k_out; p.t[1].w = k_weight; p.t[1].heads = num_k_heads;
    p.N = seq_len; p.tokens = batch * seq_len; p.eps = eps;
    p.chunks = (num_q_heads + kHeadRun - 1) / kHeadRun + (num_k_heads + kHeadRun - 1) / kHeadRun;
    const int64_t per = kThreads / (head_dim / 8);
    p.splits = (int64_t)p.tokens < 512 * per ? p.chunks : 1;
    const int64_t wgs = ((int64_t)p.tokens * p.splits + per - 1) / per;
    const bool inter = rotation == nullptr || rotation->interleaved != 0;
    const void* fn = dtype == MOSAIC_DTYPE_F32 ? pick<float>(head_dim, inter, norm != 0, false)
                                               : pick<bf16_t>(head_dim, inter, norm != 0, false);
    void* args[] = {&p};
    const unsigned grid = (unsigned)(wgs < (1 << 22) ? wgs : (1 << 22));
    return hipLaunchKernel(fn, dim3(grid), dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)) == hipSuccess
               ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

size_t mosaic_qk_norm_bwd_workspace_size(int32_t batch, int32_t seq_len, int32_t head_dim) {
    if (batch <= 0 || seq_len <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)bwd_groups((int64_t)batch * seq_len, head_dim) * 2 * head_dim * sizeof(float);
}

int mosaic_qk_norm_rotate_bwd(mosaic_bnhd grad_q, mosaic_bnhd grad_k, mosaic_bnhd q, mosaic_bnhd k, int32_t dtype,
                              int32_t batch, int32_t seq_len, int32_t num_q_heads, int32_t num_k_heads,
                              int32_t head_dim, const mosaic_rotation* rotation, const float* q_weight,
                              const float* k_weight, float eps, void* dq, void* dk, float* q_weight_grad,
                              float* k_weight_grad, void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_shape(dtype, batch, seq_len, num_q_heads, num_k_heads, head_dim)) return e;
    if (!(eps >= 0.f)) return MOSAIC_ERR_MODE;
    if (int e = check_rows(q, dtype)) return e;
    if (int e = check_rows(grad_q, dtype)) return e;
    if (dq == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (num_k_heads > 0) {
        if (int e = check_rows(k, dtype)) return e;
        if (int e = check_rows(grad_k, dtype)) return e;
        if (dk == nullptr) return MOSAIC_ERR_NULL_POINTER;
    }
    for (const void* a : {(const void*)dq, (const void*)dk}) if (!aligned(a, 16)) return MOSAIC_ERR_ALIGNMENT;
    for (const void* a : {(const void*)q_weight, (const void*)k_weight, (const void*)q_weight_grad, (const void*)k_weight_grad})
        if (!aligned(a, 4)) return MOSAIC_ERR_ALIGNMENT;
    const bool sums = q_weight_grad != nullptr || k_weight_grad != nullptr;
    if (sums && (workspace == nullptr || !aligned(workspace, 16) ||
                 workspace_bytes < mosaic_qk_norm_bwd_workspace_size(batch, seq_len, head_dim)))
        return MOSAIC_ERR_WORKSPACE;
    RotParams p{};
    if (int e = fill_rotation(p, rotation, head_dim)) return e;
    p.sign = -1.f;
    const mosaic_bnhd* xs[2] = {&q, &k};
    const mosaic_bnhd* gs[2] = {&grad_q, &grad_k};
    for (int i = 0; i < 2; ++i) {
        p.t[i].x = xs[i]->ptr; p.t[i].sb = xs[i]->stride_b; p.t[i].sn = xs[i]->stride_n; p.t[i].sh = xs[i]->stride_h;
        p.t[i].g = gs[i]->ptr; p.t[i].gsb = gs[i]->stride_b; p.t[i].gsn = gs[i]->stride_n; p.t[i].gsh = gs[i]->stride_h;
    }
    p.t[0].y = dq; p.t[0].w = q_weight; p.t[0].heads = num_q_heads;
    p.t[1].y = dk; p.t[1].w = k_weight; p.t[1].heads = num_k_heads;
    p.N = seq_len; p.tokens = batch * seq_len; p.eps = eps;
    p.partial = sums ? static_cast<float*>(workspace) : nullptr;
    const bool inter = rotation == nullptr || rotation->interleaved != 0;
    const void* fn = dtype == MOSAIC_DTYPE_F32 ? pick<float>(head_dim, inter, true, true) : pick<bf16_t>(head_dim, inter, true, true);
    const int groups = bwd_groups(p.tokens, head_dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    void* args[] = {&p};
    if (hipLaunchKernel(fn, dim3(groups), dim3(kThreads), args, 0, s) != hipSuccess) return MOSAIC_ERR_LAUNCH;
    if (!sums) return MOSAIC_OK;
    const float* part = p.partial;
    int rows = groups, D = head_dim;
    void* wargs[] = {&part, &rows, &D, &q_weight_grad, &k_weight_grad};
    return hipLaunchKernel((const void*)&wgrad_kernel, dim3(2 * head_dim / 8), dim3(kThreads), wargs, 0, s) == hipSuccess
               ? MOSAIC_OK : MOSAIC_ERR_LAUNCH;
}

}  // extern "C"
