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

// The byte of a tile that holds channels d (even) and d + 1 of token t's key or value is a sum of a part for the token and one
// for the channel. The 8 bytes of a block of 16 channels are neighbours, except for values of D = 64: two runs of 4 bytes, 64
// bytes apart.
template <int D> __device__ __forceinline__ int k_token(int t) {
  return (2 * (t >> 2) + (t & 1)) * 64 + ((t >> 1) & 1) * (D == 64 ? 8 : 4 * D);
}
template <int D> __device__ __forceinline__ int k_channel(int d) {
  const int in_lane = d % (D / 4) / 2;
  return in_lane / 16 * 512 + d / (D / 4) * 16 + in_lane % 16;
}
template <int D> __device__ __forceinline__ int v_token(int t) {
  return (t >> 2) * 16 + (D == 64 ? (t & 3) * 4 : D == 128 ? (t >> 1 & 1) * 512 + (t & 1) * 8 : (t & 3) * 512);
}
template <int D> __device__ __forceinline__ int v_channel(int d) { return Tile<D>::v + d / (D / 8) * 64 + d % (D / 8) / 2; }
template <int D> __device__ __forceinline__ int k_byte(int t, int d) { return k_token<D>(t) + k_channel<D>(d); }
template <int D> __device__ __forceinline__ int v_byte(int t, int d) { return v_token<D>(t) + v_channel<D>(d); }
// scale of block b (16 channels), the same way
template <int D> __device__ __forceinline__ int k_sf_token(int t) {
  return (2 * (t >> 2) + (t & 1)) * (D / 8) + ((t >> 1) & 1) * (D / 64);
}
template <int D> __device__ __forceinline__ int k_sf_block(int b) { return Tile<D>::k_sf + b / (D / 64) * (D / 32) + b % (D / 64); }
template <int D> __device__ __forceinline__ int k_sf_byte(int t, int b) { return k_sf_token<D>(t) + k_sf_block<D>(b); }
template <int D> __device__ __forceinline__ int v_sf_byte(int t, int b) { return Tile<D>::v_sf + b * 16 + t; }

// Tile of token slot `loc` (page * page_size + offset) and head h; pages hold page_size / 16 tiles of each head.
template <int D> __device__ __forceinline__ long long tile_at(long long page, int off, int h, int hk, int page_size) {
  return ((page * hk + h) * (page_size / kTile) + off / kTile) * Tile<D>::bytes;
}

__device__ __forceinline__ float2 decode2(uint32_t byte) {
  const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(byte & 0xFF), __NV_E2M1);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

inline int device_sms() {
  static int sms[64] = {};
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && sms[dev]) return sms[dev];
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 0 && dev < 64) sms[dev] = n;
  return n;
}

}  // namespace fp4
}  // namespace msgl
