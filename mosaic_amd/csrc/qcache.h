// qcache.h -- the layout of a key/value cache held in 8 bits, and its codes.
//
// A cache has nb blocks of bs tokens for each batch member and kv head.  Block (b, j, h) holds the
// codes of its tokens' keys and those of their values, bs * 64 bytes each, and a scale of each: the
// value of a code is code * scale.  Codes lie in the order in which a wave of the attention reads them
// as operands of v_mfma_f32_32x32x16_bf16, 16 bytes a lane and 1 KB a load, without LDS or transposing:
// a tile of 64 tokens is four such runs,
//   keys    [kt 2][dp 2][hh 2][row 32]: dims 32 dp + 16 hh .. + 15 of token 32 kt + key_of_row(row)
//   values  [kt 2][dt 2][hh 2][dim 32]: tokens 32 kt + 16 hh .. + 15, dim 32 dt + dim
// With the rows so ordered, accumulator e of lane half hh of S^T = K Q^T is token 16 hh + e, which is
// the token of element e of that lane half's operand of the product with the values.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "bsa_common.h"
#include "mosaic_bsa.h"

namespace mosaic {
namespace {

constexpr int kCodeTile = 64 * 64;   // bytes of 64 tokens' keys, or values

// Token (of 32) of row r of the keys' operand
__device__ __forceinline__ int key_of_row(int r) { return 16 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3); }

__device__ __forceinline__ int64_t block_at(const mosaic_kv_cache& c, int b, int j, int h) {
    return ((int64_t)b * c.num_blocks + j) * c.num_kv_heads + h;
}

// Four codes of a word as bf16, exactly, two to a word.
template <bool FP8>
__device__ __forceinline__ uint2 codes_bf16(uint32_t w) {
    if constexpr (FP8) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
        return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    } else {
        // a whole number below 2^8 is an fp32 number whose lower half is zero
        const uint32_t x0 = __float_as_uint((float)(int8_t)w), x1 = __float_as_uint((float)(int8_t)(w >> 8));
        const uint32_t x2 = __float_as_uint((float)(int8_t)(w >> 16)), x3 = __float_as_uint((float)((int32_t)w >> 24));
        return make_uint2(__builtin_amdgcn_perm(x1, x0, 0x07060302), __builtin_amdgcn_perm(x3, x2, 0x07060302));
    }
}

// Four codes of a word as fp32.
template <bool FP8>
__device__ __forceinline__ float4 codes_f32(uint32_t w) {
    if constexpr (FP8) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        return make_float4((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)((int32_t)w >> 24));
    }
}

// Whether a launch's threads can be counted: in 32 bits.
inline bool grid_fits(int64_t groups, int threads) { return groups < (1LL << 32) / threads; }

// Whether a cache's description can be addressed.
inline int check_cache(const mosaic_kv_cache* c) {
    if (c == nullptr) return MOSAIC_ERR_NULL_POINTER;
    if (c->k_codes == nullptr || c->v_codes == nullptr || c->k_scale == nullptr || c->v_scale == nullptr ||
        c->k_norm == nullptr || c->k_mean == nullptr)
        return MOSAIC_ERR_NULL_POINTER;
    if (c->batch <= 0 || c->num_blocks <= 0 || c->capacity <= 0) return MOSAIC_ERR_SHAPE;
    if (c->num_kv_heads <= 0 || c->num_kv_heads > 65535) return MOSAIC_ERR_HEADS;   // (a block of all heads is below 2^31 bytes)
    if (c->block_size != 64 && c->block_size != 128 && c->block_size != 256) return MOSAIC_ERR_BLOCK_SIZE;
    if (c->code_type != MOSAIC_CODE_INT8 && c->code_type != MOSAIC_CODE_E4M3) return MOSAIC_ERR_UNSUPPORTED;
    // positions of tokens, and tiles of 64 of all heads and members, are counted in 31 bits
    if ((int64_t)c->num_blocks * c->block_size > 0x7fffffff - 1024) return MOSAIC_ERR_SHAPE;
    if (c->capacity > c->num_blocks * c->block_size) return MOSAIC_ERR_SHAPE;
    if ((double)c->num_blocks * (c->block_size / 64) * c->num_kv_heads * c->batch > 2147483647.0 - 1024) return MOSAIC_ERR_SHAPE;
    auto low = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; };
    if (low(c->k_codes, 16) || low(c->v_codes, 16) || low(c->k_scale, 4) || low(c->v_scale, 4) || low(c->k_norm, 4) || low(c->k_mean, 16))
        return MOSAIC_ERR_ALIGNMENT;
    return MOSAIC_OK;
}

}  // namespace
}  // namespace mosaic
