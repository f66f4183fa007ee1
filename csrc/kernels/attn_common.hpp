// Register-tile helpers shared by the attention kernels: the dropout decision of a probability, conversions of accumulator
// tiles into matrix operands, and reductions over the lane groups that share a score row.
#pragma once
#include "common.hpp"

namespace pdt {

constexpr float LOG2E = 1.4426950408889634f;

// Dropout decision for probability (bh, q, key): a function of (seed, offset, site, micro, b*A+h, q, key) only,
// so every kernel agrees whatever its lane mapping is.  It is split in two so that the per-element cost is one
// 32-bit multiply: a strongly mixed 32-bit seed per query row (computed once per row - in the dK/dV sweeps it
// is staged in LDS), and per element  x = low24(row_seed ^ key * GOLD) * MIX24,  keep <=> x[31:16] >= thr.
// key * GOLD is a Weyl sequence over the keys; an unrolled sweep forms it with one add per element.
__device__ __forceinline__ uint32_t lowbias32(uint32_t x) {
  x ^= x >> 16; x *= 0x7feb352du; x ^= x >> 15; x *= 0x846ca68bu; x ^= x >> 16;
  return x;
}
constexpr uint32_t ATT_GOLD = 0x9E3779B9u, ATT_MIX = 0xEBCA6Bu;
__device__ __forceinline__ uint32_t attn_row_seed(const DropKey& dk, uint32_t bh, uint32_t q) {
  uint32_t x = lowbias32(q ^ dk.key.x);
  return lowbias32(x ^ (bh * 0x9E3779B9u) ^ dk.key.y ^ (dk.stream * 0x85EBCA6Bu) ^ (dk.micro * 0xC2B2AE35u));
}
// thr_hi = drop threshold << 16 (see attn_thr_hi); kmul = key * ATT_GOLD
__device__ __forceinline__ bool attn_keep(uint32_t row_seed, uint32_t kmul, uint32_t thr_hi) {
  return __umul24(row_seed ^ kmul, ATT_MIX) >= thr_hi;  // 24 x 24 -> low 32 bits: a full-rate multiply
}
__device__ __forceinline__ uint32_t attn_thr_hi(uint32_t thr) { return (thr > 65535u ? 65535u : thr) << 16; }

// The per-score arithmetic of these kernels is written on whole float4v accumulator tiles (scale + mask, subtract the
// maximum, dropout factor, dS = P * (dP - delta)).  The build switches packed fp32 instructions off (build_ext.py), so an
// operation on 4-vectors is four scalar ones; with them on, the same kernels took the same time (forward 251 / 251 us,
// fused backward 584 / 584 us at batch 1024, both builds in turn).  Pairs of results are converted with one
// v_cvt_pk_f16_f32 / v_cvt_pk_bf16_f32.
typedef float float2v __attribute__((ext_vector_type(2)));
template <typename T> struct Pk2;
template <> struct Pk2<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(2))); };
template <> struct Pk2<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(2))); };
template <typename T>
__device__ __forceinline__ int cvt_pk(float lo, float hi) {  // two fp32 -> one dword of two 16-bit values (round to nearest even)
  return __builtin_bit_cast(int, __builtin_convertvector(float2v{lo, hi}, typename Pk2<T>::type));
}
__device__ __forceinline__ float4v splat4(float v) { return float4v{v, v, v, v}; }
template <typename T>
__device__ __forceinline__ short8 pack_pair(const float4v& a, const float4v& b) {
  const int4v r = {cvt_pk<T>(a[0], a[1]), cvt_pk<T>(a[2], a[3]), cvt_pk<T>(b[0], b[1]), cvt_pk<T>(b[2], b[3])};
  return __builtin_bit_cast(short8, r);
}
__device__ __forceinline__ float quad_sum(float v) {  // sum over the 4 lane groups (lanes l, l^16, l^32, l^48)
  v += __shfl_xor(v, 16, 64);
  v += __shfl_xor(v, 32, 64);
  return v;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// sum over the 16 lanes of a DPP row (lanes sharing lane>>4); every lane of the row receives the total
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp_f<0x128>(v);  // row_ror:8
  v += dpp_f<0x124>(v);  // row_ror:4
  v += dpp_f<0x122>(v);  // row_ror:2
  v += dpp_f<0x121>(v);  // row_ror:1
  return v;
}

}  // namespace pdt
