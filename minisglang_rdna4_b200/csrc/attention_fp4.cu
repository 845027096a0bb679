// Attention over the paged K/V pool of 4 bits (kv_fp4.cuh).
#include "kv_fp4.cuh"

using namespace msgl;
using namespace msgl::fp4;

namespace {

struct Fp4Args {
  const void* q;
  void* out;
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* cu_q;
  const int32_t* lens;
  const float* k_head;
  const float* v_head;
  float* weights;
  int width, B, hq, hk, page_size, pages, window;
  float scale;
};

// A CTA for each (request, key head); rows and the heads that share the keys one after another. Softmax statistics first, then
// the probabilities again and the sum of the values.
template <typename T, int D> __global__ void __launch_bounds__(256) fp4_attention_simple_kernel(const Fp4Args a) {
  pdl_enter();
  __shared__ float qs[D], ps[256], scratch[32];
  const int b = blockIdx.x / a.hk, h = blockIdx.x % a.hk, G = a.hq / a.hk;
  const int q0 = a.cu_q[b], q_len = a.cu_q[b + 1] - q0;
  const int n = min(a.lens[b], a.width * a.page_size);
  const float kh = a.k_head != nullptr ? a.k_head[h] : 1.f, vh = a.v_head != nullptr ? a.v_head[h] : 1.f;
  auto tile_of = [&](int i) {
    const int page = min(max(a.table[(long long)b * a.width + i / a.page_size], 0), a.pages - 1);
    return a.pool + tile_at<D>(page, i % a.page_size, h, a.hk, a.page_size);
  };
  for (int r = 0; r < q_len * G; ++r) {
    const long long row = q0 + r / G;
    const int head = h * G + r % G, pos = n - q_len + r / G;
    const int hi = min(n, pos + 1), lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += 256) qs[d] = to_float(reinterpret_cast<const T*>(a.q)[(row * a.hq + head) * D + d]) * a.scale * kh;
    __syncthreads();
    auto score = [&](int i) {
      const uint8_t* tile = tile_of(i);
      const int t = i % kTile;
      float s = 0.f;
      for (int blk = 0; blk < D / 16; ++blk) {
        float part = 0.f;
        for (int d = 0; d < 16; d += 2) {
          const float2 x = decode2(tile[k_byte<D>(t, blk * 16 + d)]);
          part += qs[blk * 16 + d] * x.x + qs[blk * 16 + d + 1] * x.y;
        }
        s += part * e4m3_to_float(tile[k_sf_byte<D>(t, blk)]);
      }
      return s;
    };
    float m = -INFINITY;
    for (int i = lo + threadIdx.x; i < hi; i += 256) m = fmaxf(m, score(i));
    m = block_max(m, scratch);
    float l = 0.f;
    for (int i = lo + threadIdx.x; i < hi; i += 256) l += expf(score(i) - m);
    l = block_sum(l, scratch);
    float o = 0.f;
    for (int i0 = lo; i0 < hi; i0 += 256) {
      const int i = i0 + threadIdx.x;
      const float p = i < hi ? expf(score(i) - m) / l : 0.f;
      __syncthreads();
      ps[threadIdx.x] = p;
      if (i < hi && a.weights != nullptr) {
        const int page = min(max(a.table[(long long)b * a.width + i / a.page_size], 0), a.pages - 1);
        atomicAdd(a.weights + ((long long)page * a.hk + h) * a.page_size + i % a.page_size, p);
      }
      __syncthreads();
      if (threadIdx.x < D) {
        const int d = threadIdx.x;
        for (int k = 0; k < min(256, hi - i0); ++k) {
          const uint8_t* tile = tile_of(i0 + k);
          const int t = (i0 + k) % kTile;
          const float2 x = decode2(tile[v_byte<D>(t, d & ~1)]);
          o += ps[k] * (d & 1 ? x.y : x.x) * e4m3_to_float(tile[v_sf_byte<D>(t, d / 16)]);
        }
      }
    }
    if (threadIdx.x < D)
      reinterpret_cast<T*>(a.out)[(row * a.hq + head) * D + threadIdx.x] = from_float<T>(o * vh);
  }
}

}  // namespace

MSGL_API int msgl_attention_fp4(const void* q, void* out, const void* pool, const void* table, int width, const void* cu_q,
                                const void* lens, const void* k_head, const void* v_head, void* weights, int B, int hq, int hk, int d,
                                int page_size, int pages, int window, float scale, int dtype, cudaStream_t stream) {
  if (B <= 0) return MSGL_OK;
  if (hk <= 0 || hq % hk || (d != 64 && d != 128 && d != 256) || page_size <= 0 || page_size % kTile || (uintptr_t)pool % 16 ||
      (uintptr_t)q % 16 || (uintptr_t)out % 16 || width <= 0 || (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("paged_attention_fp4: heads of 64, 128 or 256 channels, pages of whole tiles of 16 tokens, 16-bit queries");
    return MSGL_BAD_ARG;
  }
  Fp4Args a{q, out, (const uint8_t*)pool, (const int32_t*)table, (const int32_t*)cu_q, (const int32_t*)lens, (const float*)k_head,
            (const float*)v_head, (float*)weights, width, B, hq, hk, page_size, pages, window, scale};
#define ATT(T, D) msgl_launch(fp4_attention_simple_kernel<T, D>, dim3(B * hk), dim3(256), 0, stream, a)
  if (dtype == MSGL_BF16) { if (d == 64) ATT(__nv_bfloat16, 64); else if (d == 128) ATT(__nv_bfloat16, 128); else ATT(__nv_bfloat16, 256); }
  else { if (d == 64) ATT(__half, 64); else if (d == 128) ATT(__half, 128); else ATT(__half, 256); }
#undef ATT
  MSGL_CHECK_LAUNCH("paged_attention_fp4");
  return MSGL_OK;
}
