// Layout of the paged K/V pool of 4 bits and its number format.
//
// A value is code * scale * head: an e2m1 code, an e4m3 scale for 16 neighbouring channels, an fp32 factor per key / value
// head. 16 tokens of one head are a tile of 18 D bytes: codes of the keys (8 D), of the values (8 D), scales of the keys (D), of
// the values (D). Inside, everything lies in the order in which the lanes of a warp take it as the 16 x 16 operand of a matrix
// instruction (lane 4 g + j: rows g and g + 8, columns 2 j, 2 j + 1, 2 j + 8, 2 j + 9), so that a warp fetches a tile with
// plain 16-byte loads, 512 bytes at a time, and neither transposes nor shuffles:
//   * keys (rows are tokens, columns channels): row g + 8 r is token 4 (g / 2) + 2 r + g % 2; lane j has channels j D / 4 and on.
//   * values (rows are channels, columns tokens): column pairs of lane j are tokens 4 j .. 4 j + 3; lane g has channels
//     g D / 8 and on.
// A row's order of tokens is the columns' order too, so the probabilities that one product leaves are the other's operand.
#pragma once
#include "common.cuh"
#include <cuda_fp4.h>

namespace msgl {
namespace fp4 {

constexpr int kTile = 16;                                    // tokens
template <int D> struct Tile {
  static constexpr int bytes = 18 * D, v = 8 * D, k_sf = 16 * D, v_sf = 17 * D;
};

// Byte of the tile that holds channels d (even) and d + 1 of token t's key / value; the 8 bytes of a block of 16 channels are
// neighbours, except for values of D = 64: two runs of 4 bytes, 64 bytes apart.
template <int D> __device__ __forceinline__ int k_byte(int t, int d) {
  const int g = 2 * (t >> 2) + (t & 1), r = (t >> 1) & 1, j = d / (D / 4);
  const int at = r * (D / 8) + (d % (D / 4)) / 2;
  return at / 16 * 512 + (4 * g + j) * 16 + at % 16;
}
template <int D> __device__ __forceinline__ int v_byte(int t, int d) {
  const int j = t >> 2, e = t & 3, g = d / (D / 8);
  const int at = e * (D / 16) + (d % (D / 8)) / 2;
  return Tile<D>::v + at / 16 * 512 + (4 * g + j) * 16 + at % 16;
}
// scale of block b (16 channels)
template <int D> __device__ __forceinline__ int k_sf_byte(int t, int b) {
  const int g = 2 * (t >> 2) + (t & 1), r = (t >> 1) & 1, j = b / (D / 64);
  return Tile<D>::k_sf + (4 * g + j) * (D / 32) + r * (D / 64) + b % (D / 64);
}
template <int D> __device__ __forceinline__ int v_sf_byte(int t, int b) {
  return Tile<D>::v_sf + (b * 4 + (t >> 2)) * 4 + (t & 3);
}

// Tile of token slot `loc` (page * page_size + offset) and head h; pages hold page_size / 16 tiles of each head.
template <int D> __device__ __forceinline__ long long tile_at(long long page, int off, int h, int hk, int page_size) {
  return ((page * hk + h) * (page_size / kTile) + off / kTile) * Tile<D>::bytes;
}

// 16 channels -> 8 bytes of codes and the scale. The scale is the magnitude that the largest code (6) stands for, rounded to
// e4m3 (3 bits of mantissa: what one byte for 16 values leaves); a code is the nearest of x / (scale * head), ties to the even
// one. Divisions are IEEE ones: a quotient that lies on a tie has to stay there.
__device__ __forceinline__ uint2 quantise16(const float (&x)[16], float head, uint8_t& sf) {
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    top = fmaxf(top, fabsf(x[i]));
    nan |= x[i] != x[i];
  }
  sf = nan ? 0x7F : (uint8_t)float_to_e4m3(top / (6.f * head));   // a NaN of the block shows in all of it
  const float step = e4m3_to_float(sf) * head;
  uint32_t w[2] = {0, 0};
  if (step > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i / 4] |= (uint32_t)__nv_cvt_float2_to_fp4x2(make_float2(x[2 * i] / step, x[2 * i + 1] / step), __NV_E2M1, cudaRoundNearest)
                  << (8 * (i % 4));
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float2 decode2(uint32_t byte) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(byte & 0xFF), __NV_E2M1);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace fp4
}  // namespace msgl
