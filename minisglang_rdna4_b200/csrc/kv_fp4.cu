// Rows of the paged K/V pool of 4 bits (kv_fp4.cuh): store, load, and eviction by accumulated attention weight.
#include "kv_fp4.cuh"

using namespace msgl;
using namespace msgl::fp4;

namespace {

struct RowArgs {
  const void* k;            // store: rows in; load: rows out
  const void* v;
  long long ldk, ldv;       // elements from row to row
  uint8_t* pool;            // [layers, pages, hk, page_size / 16, 18 D]
  long long layer_bytes;
  const int32_t* loc;
  const float* k_head;      // [hk] or null: 1
  const float* v_head;
  float* weights;           // store: attention weights of the slots that are written start at 0, or null
  int rows, hk, page_size, layers;
  long long slots;
};

// A thread has one block of 16 channels of a key or value: 32 bytes in, 8 bytes and a scale out. Bound: DRAM; neighbouring
// threads read neighbouring blocks of one row.
template <typename T, int D> __global__ void __launch_bounds__(256) store_fp4_kernel(const RowArgs a) {
  pdl_enter();
  constexpr int NB = D / 16;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)(id % NB);
  const long long rest = id / NB;
  const int h = (int)(rest % a.hk);
  const long long row = rest / a.hk;
  if (row >= a.rows) return;
  const bool val = blockIdx.y != 0;
  const long long loc = a.loc[row];
  (void)MSGL_OOB(loc, a.slots);
  if (loc < 0 || loc >= a.slots) return;
  const T* src = reinterpret_cast<const T*>(val ? a.v : a.k) + row * (val ? a.ldv : a.ldk) + h * D + b * 16;
  float x[16];
  {
    float lo[8], hi[8];
    load8(src, lo);
    load8(src + 8, hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x[i] = lo[i]; x[8 + i] = hi[i]; }
  }
  const float* heads = val ? a.v_head : a.k_head;
  uint8_t sf;
  const uint2 code = quantise16(x, heads != nullptr ? heads[h] : 1.f, sf);
  const long long page = loc / a.page_size;
  const int off = (int)(loc - page * a.page_size), t = off % kTile;
  uint8_t* tile = a.pool + tile_at<D>(page, off, h, a.hk, a.page_size);
  if (!val) {
    *reinterpret_cast<uint2*>(tile + k_byte<D>(t, b * 16)) = code;
    tile[k_sf_byte<D>(t, b)] = sf;
    if (b == 0 && a.weights != nullptr) a.weights[(page * a.hk + h) * a.page_size + off] = 0.f;
  } else {
    if (D == 64) {
      *reinterpret_cast<uint32_t*>(tile + v_byte<D>(t, b * 16)) = code.x;
      *reinterpret_cast<uint32_t*>(tile + v_byte<D>(t, b * 16 + 8)) = code.y;
    } else {
      *reinterpret_cast<uint2*>(tile + v_byte<D>(t, b * 16)) = code;
    }
    tile[v_sf_byte<D>(t, b)] = sf;
  }
}

// The inverse, a block of 16 channels a thread. A slot outside the pool gives zeros.
template <typename T, int D> __global__ void __launch_bounds__(256) load_fp4_kernel(const RowArgs a) {
  pdl_enter();
  constexpr int NB = D / 16;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)(id % NB);
  const long long rest = id / NB;
  const int h = (int)(rest % a.hk);
  const long long out_row = rest / a.hk;
  if (out_row >= (long long)a.rows * a.layers) return;
  const long long layer = out_row / a.rows, row = out_row - layer * a.rows;
  const bool val = blockIdx.y != 0;
  const long long loc = a.loc[row];
  (void)MSGL_OOB(loc, a.slots);
  float lo[8] = {}, hi[8] = {};
  if (loc >= 0 && loc < a.slots) {
    const long long page = loc / a.page_size;
    const int off = (int)(loc - page * a.page_size), t = off % kTile;
    const uint8_t* tile = a.pool + layer * a.layer_bytes + tile_at<D>(page, off, h, a.hk, a.page_size);
    uint2 code;
    float s;
    if (!val) {
      code = *reinterpret_cast<const uint2*>(tile + k_byte<D>(t, b * 16));
      s = e4m3_to_float(tile[k_sf_byte<D>(t, b)]) * (a.k_head != nullptr ? a.k_head[h] : 1.f);
    } else {
      if (D == 64) {
        code.x = *reinterpret_cast<const uint32_t*>(tile + v_byte<D>(t, b * 16));
        code.y = *reinterpret_cast<const uint32_t*>(tile + v_byte<D>(t, b * 16 + 8));
      } else {
        code = *reinterpret_cast<const uint2*>(tile + v_byte<D>(t, b * 16));
      }
      s = e4m3_to_float(tile[v_sf_byte<D>(t, b)]) * (a.v_head != nullptr ? a.v_head[h] : 1.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = decode2(code.x >> (8 * i)), q = decode2(code.y >> (8 * i));
      lo[2 * i] = p.x * s; lo[2 * i + 1] = p.y * s;
      hi[2 * i] = q.x * s; hi[2 * i + 1] = q.y * s;
    }
  }
  T* dst = reinterpret_cast<T*>(const_cast<void*>(val ? a.v : a.k)) + (out_row * a.hk + h) * D + b * 16;
  store8(dst, lo);
  store8(dst + 8, hi);
}

// ---- eviction --------------------------------------------------------------------------
struct EvictArgs {
  uint8_t* pool;
  long long layer_bytes;
  float* weights;           // [layers, pages, hk, page_size]
  long long layer_weights;
  const int32_t* table;     // [requests, width]
  const int32_t* new_table; // [requests, new_width]
  int32_t* kept;            // [layers, requests, hk, budget]
  int32_t* new_lens;        // [requests]
  const int32_t* lens;
  int width, new_width, requests, hk, page_size, pages, budget, recent, sinks;
};

__device__ __forceinline__ int page_of(const EvictArgs& a, const int32_t* table, int width, int b, int i) {
  const int col = min(i / a.page_size, width - 1);
  const int page = table[(long long)b * width + col];
  (void)MSGL_OOB(page, a.pages);
  return min(max(page, 0), a.pages - 1);
}

// Larger weight, larger key; both zeros are one key; NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// A CTA for each (layer, request, head): the key of the last weight that stays by a radix search (four digits of 8 bits), then
// the tokens above it, and of those at it the first ones, in their order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
  pdl_enter();
  __shared__ int hist[256];
  __shared__ int warp_sum_above[32], warp_sum_tie[32];
  __shared__ uint32_t s_digit;
  __shared__ int s_rank;
  const int h = blockIdx.x % a.hk, b = blockIdx.x / a.hk % a.requests, layer = blockIdx.x / a.hk / a.requests;
  const int n = min(max(a.lens[b], 0), a.width * a.page_size);
  int32_t* kept = a.kept + (long long)blockIdx.x * a.budget;
  if (layer == 0 && h == 0 && threadIdx.x == 0) a.new_lens[b] = min(n, a.budget);
  if (n <= a.budget) {
    for (int i = threadIdx.x; i < a.budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int lo = a.sinks, hi = n - a.recent, need = a.budget - a.sinks - a.recent;   // candidates [lo, hi): more than need
  const float* weights = a.weights + layer * a.layer_weights;
  auto key_of = [&](int i) {
    const long long page = page_of(a, a.table, a.width, b, i);
    return weight_key(weights[(page * a.hk + h) * a.page_size + i % a.page_size]);
  };
  uint32_t bound = 0, mask = 0;
  int rank = need;          // of the bound among the keys that share its digits so far, from the largest, from 1
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + threadIdx.x; i < hi; i += kSelThreads) {
        const uint32_t key = key_of(i);
        if ((key & mask) == bound) atomicAdd(&hist[key >> shift & 255], 1);
      }
      __syncthreads();
      if (threadIdx.x < 32) {
        // lane l has digits 255 - 8 l and down
        int sum = 0;
        for (int q = 0; q < 8; ++q) sum += hist[255 - 8 * threadIdx.x - q];
        int incl = sum;
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, incl, o);
          if ((int)threadIdx.x >= o) incl += up;
        }
        int before = incl - sum;
        if (before < rank && rank <= incl) {
          for (int q = 0; q < 8; ++q) {
            const int c = hist[255 - 8 * threadIdx.x - q];
            if (rank <= before + c) { s_digit = 255 - 8 * threadIdx.x - q; s_rank = rank - before; break; }
            before += c;
          }
        }
      }
      __syncthreads();
      bound |= s_digit << shift;
      mask |= 255u << shift;
      rank = s_rank;
      __syncthreads();
    }
  }
  // tokens in order: what is above the bound, and the first `rank` at it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < a.sinks; i += kSelThreads) kept[i] = i;
  for (int i = threadIdx.x; i < a.recent; i += kSelThreads) kept[a.budget - a.recent + i] = hi + i;
  int above = 0, ties = 0;          // so far
  for (int i0 = lo; i0 < hi && need > 0; i0 += kSelThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t key = i < hi ? key_of(i) : 0;
    const bool up = i < hi && key > bound, tie = i < hi && key == bound;
    const uint32_t up_bits = __ballot_sync(0xffffffffu, up), tie_bits = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) { warp_sum_above[warp] = __popc(up_bits); warp_sum_tie[warp] = __popc(tie_bits); }
    __syncthreads();
    int ua = above, ta = ties, uall = 0, tall = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) { ua += warp_sum_above[w]; ta += warp_sum_tie[w]; }
      uall += warp_sum_above[w];
      tall += warp_sum_tie[w];
    }
    ua += __popc(up_bits & ((1u << lane) - 1));
    ta += __popc(tie_bits & ((1u << lane) - 1));
    if (up || (tie && ta < rank)) kept[lo + ua + min(ta, rank)] = i;
    above += uall;
    ties += tall;
    __syncthreads();
  }
}

// A warp for each tile of 16 rows that stay: every lane collects its own bytes of the new tile. Slots behind the last row keep
// what they hold.
template <int D> __global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a, int tiles, long long units) {
  pdl_enter();
  const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (id >= units) return;
  const int tile = (int)(id % tiles);
  const long long unit = id / tiles;
  const int h = (int)(unit % a.hk), b = (int)(unit / a.hk % a.requests);
  const long long layer = unit / a.hk / a.requests;
  const int m = a.new_lens[b];
  const int rows = min(kTile, m - tile * kTile);
  if (rows <= 0) return;
  uint8_t* pool = a.pool + layer * a.layer_bytes;
  float* weights = a.weights + layer * a.layer_weights;
  // lane t: where row t comes from
  long long from = 0;
  int t_src = 0;
  const int to_off = tile * kTile % a.page_size;
  const long long to_page = page_of(a, a.new_table, a.new_width, b, tile * kTile);
  if (lane < rows) {
    const int i = a.kept[unit * a.budget + tile * kTile + lane];
    const int off = i % a.page_size;
    const long long page = page_of(a, a.table, a.width, b, i);
    from = tile_at<D>(page, off, h, a.hk, a.page_size);
    t_src = off % kTile;
    weights[(to_page * a.hk + h) * a.page_size + to_off + lane] = weights[(page * a.hk + h) * a.page_size + off];
  }
  uint8_t* to = pool + tile_at<D>(to_page, to_off, h, a.hk, a.page_size);
  for (int t = 0; t < rows; ++t) {
    const uint8_t* src = pool + __shfl_sync(0xffffffffu, from, t);
    const int ts = __shfl_sync(0xffffffffu, t_src, t);
    for (int i = lane; i < D / 4; i += 32) {      // 4 bytes a lane
      const int d = i % (D / 8) * 8;
      const bool val = i >= D / 8;
      const int s = val ? v_byte<D>(ts, d) : k_byte<D>(ts, d), e = val ? v_byte<D>(t, d) : k_byte<D>(t, d);
      *reinterpret_cast<uint32_t*>(to + e) = *reinterpret_cast<const uint32_t*>(src + s);
    }
    for (int i = lane; i < D / 8; i += 32) {
      const int blk = i % (D / 16);
      const bool val = i >= D / 16;
      to[val ? v_sf_byte<D>(t, blk) : k_sf_byte<D>(t, blk)] = src[val ? v_sf_byte<D>(ts, blk) : k_sf_byte<D>(ts, blk)];
    }
  }
}

bool shape_ok(int hk, int d, int page_size, const void* pool, const char* what) {
  if (hk > 0 && (d == 64 || d == 128 || d == 256) && page_size > 0 && page_size % kTile == 0 && (uintptr_t)pool % 16 == 0) return true;
  msgl_set_error_text(what);
  return false;
}

}  // namespace

MSGL_API int msgl_store_fp4(const void* k, const void* v, long long ldk, long long ldv, void* pool, const void* loc, const void* k_head,
                            const void* v_head, void* weights, int rows, int hk, int d, int page_size, long long pages, int dtype,
                            cudaStream_t stream) {
  if (rows <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pool, "store_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens"))
    return MSGL_BAD_ARG;
  if (ldk % 8 || ldv % 8 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("store_kv_fp4: 16-bit rows on 16-byte boundaries");
    return MSGL_BAD_ARG;
  }
  RowArgs a{k, v, ldk, ldv, (uint8_t*)pool, 0, (const int32_t*)loc, (const float*)k_head, (const float*)v_head, (float*)weights,
            rows, hk, page_size, 1, pages * page_size};
  const long long threads = (long long)rows * hk * (d / 16);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
#define STORE(T, D) msgl_launch(store_fp4_kernel<T, D>, grid, dim3(256), 0, stream, a)
  if (dtype == MSGL_BF16) { if (d == 64) STORE(__nv_bfloat16, 64); else if (d == 128) STORE(__nv_bfloat16, 128); else STORE(__nv_bfloat16, 256); }
  else { if (d == 64) STORE(__half, 64); else if (d == 128) STORE(__half, 128); else STORE(__half, 256); }
#undef STORE
  MSGL_CHECK_LAUNCH("store_kv_fp4");
  return MSGL_OK;
}

MSGL_API int msgl_load_fp4(const void* pool, long long layer_bytes, int layers, const void* loc, const void* k_head, const void* v_head,
                           void* k, void* v, int rows, int hk, int d, int page_size, long long pages, int dtype, cudaStream_t stream) {
  if (rows <= 0 || layers <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pool, "load_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens"))
    return MSGL_BAD_ARG;
  if (dtype != MSGL_BF16 && dtype != MSGL_F16) {
    msgl_set_error_text("load_kv_fp4: rows of 16 bits");
    return MSGL_BAD_ARG;
  }
  RowArgs a{k, v, 0, 0, (uint8_t*)const_cast<void*>(pool), layer_bytes, (const int32_t*)loc, (const float*)k_head,
            (const float*)v_head, nullptr, rows, hk, page_size, layers, pages * page_size};
  const long long threads = (long long)rows * layers * hk * (d / 16);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
#define LOAD(T, D) msgl_launch(load_fp4_kernel<T, D>, grid, dim3(256), 0, stream, a)
  if (dtype == MSGL_BF16) { if (d == 64) LOAD(__nv_bfloat16, 64); else if (d == 128) LOAD(__nv_bfloat16, 128); else LOAD(__nv_bfloat16, 256); }
  else { if (d == 64) LOAD(__half, 64); else if (d == 128) LOAD(__half, 128); else LOAD(__half, 256); }
#undef LOAD
  MSGL_CHECK_LAUNCH("load_kv_fp4");
  return MSGL_OK;
}

MSGL_API int msgl_evict_fp4(void* pool, long long layer_bytes, void* weights, long long layer_weights, int layers, const void* table,
                            int width, const void* new_table, int new_width, const void* lens, void* kept, void* new_lens,
                            int requests, int hk, int d, int page_size, int pages, int budget, int recent, int sinks,
                            cudaStream_t stream) {
  if (requests <= 0 || layers <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pool, "evict_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens"))
    return MSGL_BAD_ARG;
  if (budget <= 0 || recent < 0 || sinks < 0 || recent + sinks > budget || width <= 0 ||
      (long long)new_width * page_size < budget) {
    msgl_set_error_text("evict_kv_fp4: recent + sinks <= budget, and new pages for the budget");
    return MSGL_BAD_ARG;
  }
  EvictArgs a{(uint8_t*)pool, layer_bytes, (float*)weights, layer_weights, (const int32_t*)table, (const int32_t*)new_table,
              (int32_t*)kept, (int32_t*)new_lens, (const int32_t*)lens, width, new_width, requests, hk, page_size, pages, budget,
              recent, sinks};
  const long long units = (long long)layers * requests * hk;
  msgl_launch(evict_select_kernel, dim3((unsigned)units), dim3(kSelThreads), 0, stream, a);
  MSGL_CHECK_LAUNCH("evict_select");
  const int tiles = (budget + kTile - 1) / kTile;
  const dim3 grid((unsigned)((units * tiles + 7) / 8));
#define MOVE(D) msgl_launch(evict_move_kernel<D>, grid, dim3(256), 0, stream, a, tiles, units* tiles)
  if (d == 64) MOVE(64); else if (d == 128) MOVE(128); else MOVE(256);
#undef MOVE
  MSGL_CHECK_LAUNCH("evict_move");
  return MSGL_OK;
}
