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
  int rows, hk, per;        // per: tiles of a page
  uint32_t per_magic;       // 2^32 / per, rounded up: i / per = (i * per_magic) >> 32 while i * per < 2^32
  long long slots;
};

// A thread has 8 channels of a key and of its value (16-byte accesses; D / 8 threads for a row and head) in U rows that follow
// each other, so that their loads are under way at once: four where the rows fill the GPU all the same, else one. B200, us, store
// and load with one row a thread and with four: 64 rows of 8 heads of 128 6.2, 13.8; 8192 rows 41.8, 35.7 (with a key or value a
// thread; both in one thread now 27.8, of 64 rows 4.1).
template <int D, int U> struct Place {
  int h, c, row0;           // c: channels 8 c .. 8 c + 7
  int code_at[2], sf_at[2]; // the channels' part of where they lie in a tile, of keys and of values
  __device__ __forceinline__ Place(const RowArgs& a) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, items = (D / 8) * a.hk;
    const uint32_t row = id / items, item = id - row * items;
    row0 = (int)row * U;
    c = (int)(item % (D / 8));
    h = (int)(item / (D / 8));
    code_at[0] = k_channel<D>(8 * c);
    code_at[1] = v_channel<D>(8 * c);
    sf_at[0] = k_sf_block<D>(c / 2);
    sf_at[1] = v_sf_byte<D>(0, c / 2);
  }
};
// Tile of a slot, the slot's place in an [pages, hk, page] array, and its token in the tile.
template <int D> __device__ __forceinline__ uint8_t* tile_of(const RowArgs& a, int loc, int h, int& t, long long& at) {
  const int tile = loc / kTile, page = a.per == 1 ? tile : (int)__umulhi((uint32_t)tile, a.per_magic);
  t = loc % kTile;
  const long long first = ((long long)page * a.hk + h) * a.per + (tile - page * a.per);
  at = first * kTile + t;
  return a.pool + first * Tile<D>::bytes;
}

template <typename T> __device__ __forceinline__ float magnitude(uint32_t bits);
template <> __device__ __forceinline__ float magnitude<__nv_bfloat16>(uint32_t bits) { return __uint_as_float(bits << 16); }
template <> __device__ __forceinline__ float magnitude<__half>(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }

// 8 channels -> 4 bytes of codes, and the scale of their block, whose other half the neighbouring lane has. The scale is what
// the largest code (6) needs to stand for the block's largest magnitude, rounded to e4m3 (3 bits of mantissa: what one byte
// for 16 values leaves); a code is the nearest of x / (scale * head), ties to the even one. A quotient on a tie has to stay
// there, so quotients are rounded as an IEEE division rounds them: one reciprocal for the block, and for each x the product
// with it and one correction by its remainder (P. Markstein, IBM J. Res. Dev. 34, 1990). A block that saturates, whose products
// may overflow, divides. The magnitudes are compared as integers, in pairs: a NaN is then the largest, and it
// shows in all of its block. All lanes of the warp call it.
template <typename T> __device__ __forceinline__ uint32_t quantise8(const Vec8<T>& raw, float head, uint8_t& sf) {
  uint32_t top2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top2 = __vmaxu2(top2, reinterpret_cast<const uint32_t*>(&raw)[i] & 0x7FFF7FFFu);
  top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
  const float top = magnitude<T>(max(top2 & 0xFFFFu, top2 >> 16));
  sf = top != top ? 0x7F : (uint8_t)float_to_e4m3(top / (6.f * head));
  const float step = e4m3_to_float(sf) * head;
  uint32_t w = 0;
  if (step > 0.f) {
    const float back = 1.f / step;
    auto over = [&](float x) {
      const float q = x * back;
      return fmaf(fmaf(-q, step, x), back, q);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = to_float2(raw.v[i]);
      const float2 q = sf < 0x7E ? make_float2(over(x.x), over(x.y)) : make_float2(x.x / step, x.y / step);
      w |= (uint32_t)__nv_cvt_float2_to_fp4x2(q, __NV_E2M1, cudaRoundNearest) << (8 * i);
    }
  }
  return w;
}

// Floor: the 32 bytes in and 9 out of a thread and row. Bound: the chain from a row's loads over its scale, quotients, rounding and
// packing to writes of 4 bytes (a value's in 8 sectors of 32): issue slots 64 % busy, the ALU pipe 53 %, neither full. 8192 rows of 8
// heads of 128 take 17.5 us, 2.5 TB/s.
template <typename T, int D, int U> __global__ void __launch_bounds__(256) store_fp4_kernel(const RowArgs a) {
  const Place<D, U> p(a);
  pdl_enter();
  const bool any = p.row0 < a.rows;
  Vec8<T> raw[U][2];
  int loc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = p.row0 + u;
    loc[u] = -1;
    if (row < a.rows) {
      loc[u] = a.loc[row];
      if (loc[u] >= 0) (void)MSGL_OOB(loc[u], a.slots);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      *reinterpret_cast<uint4*>(&raw[u][w]) = make_uint4(0, 0, 0, 0);
      if (row < a.rows)
        raw[u][w] = *reinterpret_cast<const Vec8<T>*>(reinterpret_cast<const T*>(w ? a.v : a.k) + row * (w ? a.ldv : a.ldk) + p.h * D + p.c * 8);
    }
  }
  const float head[2] = {any && a.k_head != nullptr ? a.k_head[p.h] : 1.f, any && a.v_head != nullptr ? a.v_head[p.h] : 1.f};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t code[2];
    uint8_t sf[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) code[w] = quantise8<T>(raw[u][w], head[w], sf[w]);
    if (loc[u] < 0 || loc[u] >= a.slots) continue;
    int t;
    long long at;
    uint8_t* tile = tile_of<D>(a, loc[u], p.h, t, at);
    *reinterpret_cast<uint32_t*>(tile + p.code_at[0] + k_token<D>(t)) = code[0];
    *reinterpret_cast<uint32_t*>(tile + p.code_at[1] + v_token<D>(t)) = code[1];
    if (!(p.c & 1)) {
      tile[p.sf_at[0] + k_sf_token<D>(t)] = sf[0];
      tile[p.sf_at[1] + t] = sf[1];
    }
    if (p.c == 0 && a.weights != nullptr) a.weights[at] = 0.f;
  }
}

// The inverse; code * scale is exact, the head's factor is applied in fp32 ahead of it. A slot outside the pool gives zeros.
// Bound: the 32 bytes that a thread writes for a row: 98 thousand rows of 8 heads of 128 95 us, 5.4 TB/s. blockIdx.y: layer.
template <typename T, int D, int U> __global__ void __launch_bounds__(256) load_fp4_kernel(const RowArgs a) {
  const Place<D, U> p(a);
  pdl_enter();
  if (p.row0 >= a.rows) return;
  const float head[2] = {a.k_head != nullptr ? a.k_head[p.h] : 1.f, a.v_head != nullptr ? a.v_head[p.h] : 1.f};
  const long long layer = (long long)blockIdx.y * a.layer_bytes;
  uint32_t code[U][2];
  uint8_t sf[U][2];
  int loc[U];
#pragma unroll
  for (int u = 0; u < U; ++u) loc[u] = a.loc[min(p.row0 + u, a.rows - 1)];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    code[u][0] = code[u][1] = 0;
    sf[u][0] = sf[u][1] = 0;
    if (loc[u] >= 0) (void)MSGL_OOB(loc[u], a.slots);
    if (loc[u] < 0 || loc[u] >= a.slots) continue;
    int t;
    long long at;
    const uint8_t* tile = tile_of<D>(a, loc[u], p.h, t, at) + layer;
    code[u][0] = *reinterpret_cast<const uint32_t*>(tile + p.code_at[0] + k_token<D>(t));
    code[u][1] = *reinterpret_cast<const uint32_t*>(tile + p.code_at[1] + v_token<D>(t));
    sf[u][0] = tile[p.sf_at[0] + k_sf_token<D>(t)];
    sf[u][1] = tile[p.sf_at[1] + t];
  }
  const long long to = (((long long)blockIdx.y * a.rows + p.row0) * a.hk + p.h) * D + p.c * 8;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (p.row0 + u >= a.rows) break;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float s = e4m3_to_float(sf[u][w]) * head[w];
      Vec8<T> y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = decode2(code[u][w] >> (8 * i));
        y.v[i] = Pack2<T>::make(x.x * s, x.y * s);
      }
      *reinterpret_cast<Vec8<T>*>(reinterpret_cast<T*>(const_cast<void*>(w ? a.v : a.k)) + to + (long long)u * a.hk * D) = y;
    }
  }
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
  int per;                  // tiles of a page
  uint32_t per_magic;       // 2^32 / per, rounded up
  int wide;                 // four weights may be read at once
  int layers, by_length;
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

constexpr uint32_t kZeroKey = 0x80000000u;
constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048, kCopies = 4;
constexpr int kKeysInShared = 49000;   // beside the bins, in the 227 KB of a CTA

// A CTA for each (layer, request, head): the key of the last weight that stays by a radix search of three digits (11, 11, 10
// bits), then the tokens above it, and of those at it the first ones, in their order: each warp counts and then writes a share
// of the tokens. KEPT: the keys stay in shared memory; otherwise (requests that are too long for it) every pass reads them
// again. The few bins of the first digit that the weights of a request fall into are what lanes wait for: there are four copies of
// them, and zeros (tokens that nothing has looked at yet) are counted in registers. 384 requests' heads of 12 to 40 thousand
// tokens 64 us, one CTA an SM (73 in the order of the batch; the longest first, the last wave is short); reading the weights in every
// pass, in four digits of 8 bits, 298; digits of 8, 12 and 12 bits with a copy for each lane 77 for 73.
template <bool KEPT> __global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const EvictArgs a, int longest) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ int hist[kCopies][kBins];
  __shared__ int chunk[kSelWarps], sum_above[kSelWarps], sum_tie[kSelWarps];
  __shared__ int s_digit, s_rank;
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int h = blockIdx.x % a.hk, b = blockIdx.x / a.hk % a.requests, layer = blockIdx.x / a.hk / a.requests;
  if (a.by_length) {        // more CTAs than run at once: the longest requests' first (a warp ranks them)
    __shared__ int s_b;
    const int per = a.hk * a.layers, want = blockIdx.x / per, len = lane < a.requests ? a.lens[lane] : 0;
    int rank = 0;
    for (int i = 0; i < a.requests; ++i) {
      const int other = __shfl_sync(0xffffffffu, len, i);
      rank += other > len || (other == len && i < lane);
    }
    if (warp == 0 && lane < a.requests && rank == want) s_b = lane;
    __syncthreads();
    b = s_b;
    layer = blockIdx.x % per / a.hk;
  }
  const int unit = (layer * a.requests + b) * a.hk + h;
  const int n = min(max(a.lens[b], 0), a.width * a.page_size);
  const bool in_shared = KEPT && n <= longest;     // a request that is longer than the caller said reads its weights in every pass
  int32_t* kept = a.kept + (long long)unit * a.budget;
  if (layer == 0 && h == 0 && threadIdx.x == 0) a.new_lens[b] = min(n, a.budget);
  if (n <= a.budget) {
    for (int i = threadIdx.x; i < a.budget; i += kSelThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const int lo = a.sinks, hi = n - a.recent, need = a.budget - a.sinks - a.recent;   // candidates [lo, hi): more than need
  for (int i = threadIdx.x; i < a.sinks; i += kSelThreads) kept[i] = i;
  for (int i = threadIdx.x; i < a.recent; i += kSelThreads) kept[a.budget - a.recent + i] = hi + i;
  if (need == 0) return;
  const float* weights = a.weights + layer * a.layer_weights;
  const int32_t* table = a.table + (long long)b * a.width;
  auto column = [&](int i) { return a.per == 1 ? i >> 4 : (int)__umulhi((uint32_t)i >> 4, a.per_magic); };     // i / page_size
  // Four tokens at a time, i a multiple of four: all in one page. Key 0 (no weight has it, and no digit of one begins as it does)
  // stands for a token that is no candidate.
  const int lo4 = lo & ~3;
  auto read4 = [&](int i, int col, int page) {
    (void)MSGL_OOB(page, a.pages);
    page = min(max(page, 0), a.pages - 1);
    const float* at = weights + ((long long)page * a.hk + h) * a.page_size + i - col * a.page_size;
    const float4 w = a.wide ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
    uint4 k = make_uint4(weight_key(w.x), weight_key(w.y), weight_key(w.z), weight_key(w.w));
    if (i < lo || i + 4 > hi) {
      if (i < lo || i >= hi) k.x = 0;
      if (i + 1 < lo || i + 1 >= hi) k.y = 0;
      if (i + 2 < lo || i + 2 >= hi) k.z = 0;
      if (i + 3 < lo || i + 3 >= hi) k.w = 0;
    }
    return k;
  };
  auto keys4 = [&](int i) { return in_shared ? *reinterpret_cast<const uint4*>(keys + i) : read4(i, column(i), table[column(i)]); };
  for (int i = threadIdx.x; i < kCopies * kBins; i += kSelThreads) hist[0][i] = 0;
  __syncthreads();
  uint32_t bound = 0, mask = 0;
  int rank = need;          // of the bound among the keys that share its digits so far, from the largest, from 1
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const uint32_t ones = digit == 2 ? 1023u : 2047u;
    if (digit == 0) {
      constexpr int U = 4;  // loads under way at once
      int zeros = 0;
      for (int i0 = lo4 + 4 * (int)threadIdx.x; i0 < hi; i0 += 4 * U * kSelThreads) {
        uint4 key[U];
        int page[U];
#pragma unroll
        for (int u = 0; u < U; ++u) page[u] = table[column(min(i0 + 4 * u * kSelThreads, hi - 1))];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = min(i0 + 4 * u * kSelThreads, (hi - 1) & ~3);
          key[u] = read4(i, column(i), page[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + 4 * u * kSelThreads >= hi) break;
          if (in_shared) *reinterpret_cast<uint4*>(keys + i0 + 4 * u * kSelThreads) = key[u];
          auto count = [&](uint32_t k) {
            if (k == kZeroKey) ++zeros;
            else if (k != 0) atomicAdd(&hist[lane % kCopies][k >> 21], 1);
          };
          count(key[u].x);
          count(key[u].y);
          count(key[u].z);
          count(key[u].w);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) zeros += __shfl_xor_sync(0xffffffffu, zeros, o);
      if (lane == 0 && zeros > 0) atomicAdd(&hist[0][kZeroKey >> 21], zeros);
    } else {
      for (int i = lo4 + 4 * (int)threadIdx.x; i < hi; i += 4 * kSelThreads) {
        const uint4 k = keys4(i);
        auto count = [&](uint32_t key) {
          if ((key & mask) == bound) atomicAdd(&hist[lane % kCopies][key >> shift & ones], 1);
        };
        count(k.x);
        count(k.y);
        count(k.z);
        count(k.w);
      }
    }
    __syncthreads();
    // the largest digits first: thread t has kBins / kSelThreads of them
    constexpr int PER = kBins / kSelThreads;
    int mine[PER], sum = 0;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int bin = kBins - 1 - PER * (int)threadIdx.x - q;
      mine[q] = 0;
#pragma unroll
      for (int k = 0; k < kCopies; ++k) { mine[q] += hist[k][bin]; hist[k][bin] = 0; }
      sum += mine[q];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) chunk[warp] = incl;
    __syncthreads();
    const int before_warps = __reduce_add_sync(0xffffffffu, lane < warp ? chunk[lane] : 0);
    int before = before_warps + incl - sum;
    if (before < rank && rank <= before + sum) {
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        if (before < rank && rank <= before + mine[q]) { s_digit = kBins - 1 - PER * (int)threadIdx.x - q; s_rank = rank - before; }
        before += mine[q];
      }
    }
    __syncthreads();
    bound |= (uint32_t)s_digit << shift;
    mask |= ones << shift;
    rank = s_rank;
  }
  // what is above the bound, and the first `rank` at it
  const int share = ((hi - lo4 + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
  const int i0 = min(lo4 + warp * share, hi), i1 = min(i0 + share, hi);
  int above = 0, ties = 0;
  for (int i = i0 + 4 * lane; i < i1; i += 128) {
    const uint4 k = keys4(i);
    above += (k.x > bound) + (k.y > bound) + (k.z > bound) + (k.w > bound);
    ties += (k.x == bound) + (k.y == bound) + (k.z == bound) + (k.w == bound);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    above += __shfl_xor_sync(0xffffffffu, above, o);
    ties += __shfl_xor_sync(0xffffffffu, ties, o);
  }
  if (lane == 0) { sum_above[warp] = above; sum_tie[warp] = ties; }
  __syncthreads();
  above = __reduce_add_sync(0xffffffffu, lane < warp ? sum_above[lane] : 0);
  ties = __reduce_add_sync(0xffffffffu, lane < warp ? sum_tie[lane] : 0);
  for (int i = i0 + 4 * lane; i - 4 * lane < i1; i += 128) {
    const uint4 k = i < i1 ? keys4(i) : make_uint4(0, 0, 0, 0);
    if (!__any_sync(0xffffffffu, k.x >= bound || k.y >= bound || k.z >= bound || k.w >= bound)) continue;
    const int mine = (k.x > bound) + (k.y > bound) + (k.z > bound) + (k.w > bound) +
                     ((k.x == bound) + (k.y == bound) + (k.z == bound) + (k.w == bound) << 16);
    int incl = mine;         // above the bound, and at it, in 16 bits each
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    int ua = above + (incl - mine & 0xFFFF), ta = ties + (incl - mine >> 16);
    auto put = [&](uint32_t key, int t) {
      if (key > bound || (key == bound && ta < rank)) kept[lo + ua + min(ta, rank)] = t;
      ua += key > bound;
      ta += key == bound;
    };
    put(k.x, i);
    put(k.y, i + 1);
    put(k.z, i + 2);
    put(k.w, i + 3);
    const int all = __shfl_sync(0xffffffffu, incl, 31);
    above += all & 0xFFFF;
    ties += all >> 16;
  }
}

// A warp for each tile of 16 rows that stay: every lane collects its own bytes of the new tile, all loads ahead of the stores.
// Slots behind the last row keep what they hold. Bound: DRAM sectors of 32 bytes, of which rows that lie far apart use part: a
// row's 144 bytes (D = 128) lie in 15 sectors. 786 thousand rows' heads out of ten times as many 98 us, 615 MB from and to DRAM (6.3
// TB/s); a row at a time, its bytes over the lanes, 154.
template <int D> __global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a, int tiles, long long units) {
  pdl_enter();
  const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  if (id >= units) return;
  const int unit = (int)(id / tiles), tile = (int)(id - (long long)unit * tiles);
  const int h = unit % a.hk, b = unit / a.hk % a.requests;
  const long long layer = unit / a.hk / a.requests;
  const int m = a.new_lens[b];
  const int rows = min(kTile, m - tile * kTile);
  if (rows <= 0) return;
  uint8_t* pool = a.pool + layer * a.layer_bytes;
  float* weights = a.weights + layer * a.layer_weights;
  // lane t: where row t comes from, as (tile of the pool) * 16 + row of the tile; rows that are not there come from row 0's place
  const int to_off = tile * kTile % a.page_size;
  const int to_page = a.new_table[(long long)b * a.new_width + tile * kTile / a.page_size];
  (void)MSGL_OOB(to_page, a.pages);
  if (to_page < 0 || to_page >= a.pages) return;   // nobody's page: as the store skips a slot outside the pool
  long long from;
  {
    const int i = a.kept[(long long)unit * a.budget + tile * kTile + min(lane, rows - 1)];
    const int off = i % a.page_size;
    const long long page = page_of(a, a.table, a.width, b, i);
    from = ((page * a.hk + h) * (a.page_size / kTile) + off / kTile) * kTile + off % kTile;
    if (lane < rows) weights[((long long)to_page * a.hk + h) * a.page_size + to_off + lane] = weights[(page * a.hk + h) * a.page_size + off];
  }
  uint8_t* to = pool + tile_at<D>(to_page, to_off, h, a.hk, a.page_size);
  auto source = [&](int t, int& ts) {
    const long long f = __shfl_sync(0xffffffffu, from, t);
    ts = (int)(f % kTile);
    return pool + f / kTile * Tile<D>::bytes;
  };
  // keys: rows g and g + 8 of the operand, D / 8 bytes and D / 64 scales of each
  constexpr int KW = D / 32, SW = D / 64;
  uint32_t k[2][KW];
  uint8_t ks[2][SW];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    int ts;
    const uint8_t* src = source(4 * (g >> 1) + 2 * r + (g & 1), ts);
    if (D == 64) *reinterpret_cast<uint2*>(k[r]) = *reinterpret_cast<const uint2*>(src + k_byte<D>(ts, j * (D / 4)));
    else
#pragma unroll
      for (int w = 0; w < KW; w += 4)
        *reinterpret_cast<uint4*>(k[r] + w) = *reinterpret_cast<const uint4*>(src + k_byte<D>(ts, j * (D / 4) + 8 * w));
#pragma unroll
    for (int i = 0; i < SW; ++i) ks[r][i] = src[k_sf_byte<D>(ts, j * SW + i)];
  }
  // values: tokens 4 j .. 4 j + 3, D / 16 bytes of each; scales of the lane's blocks (D = 64: lanes of even g)
  constexpr int VW = D / 64, VB = D == 256 ? 2 : 1;
  uint32_t v[4][VW];
  uint8_t vs[4][VB];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    int ts;
    const uint8_t* src = source(4 * j + e, ts);
    const uint8_t* p = src + v_byte<D>(ts, g * (D / 8));
    if (D == 64) v[e][0] = *reinterpret_cast<const uint32_t*>(p);
    else if (D == 128) *reinterpret_cast<uint2*>(v[e]) = *reinterpret_cast<const uint2*>(p);
    else *reinterpret_cast<uint4*>(v[e]) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < VB; ++i) vs[e][i] = src[v_sf_byte<D>(ts, D == 64 ? g >> 1 : g * VB + i)];
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = 4 * (g >> 1) + 2 * r + (g & 1);
    if (t >= rows) continue;
    if (D == 64) *reinterpret_cast<uint2*>(to + k_byte<D>(t, j * (D / 4))) = *reinterpret_cast<uint2*>(k[r]);
    else
#pragma unroll
      for (int w = 0; w < KW; w += 4)
        *reinterpret_cast<uint4*>(to + k_byte<D>(t, j * (D / 4) + 8 * w)) = *reinterpret_cast<uint4*>(k[r] + w);
#pragma unroll
    for (int i = 0; i < SW; ++i) to[k_sf_byte<D>(t, j * SW + i)] = ks[r][i];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int t = 4 * j + e;
    if (t >= rows) continue;
    uint8_t* p = to + v_byte<D>(t, g * (D / 8));
    if (D == 64) *reinterpret_cast<uint32_t*>(p) = v[e][0];
    else if (D == 128) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v[e]);
    else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v[e]);
    if (D != 64 || !(g & 1))
#pragma unroll
      for (int i = 0; i < VB; ++i) to[v_sf_byte<D>(t, D == 64 ? g >> 1 : g * VB + i)] = vs[e][i];
  }
}

bool shape_ok(int hk, int d, int page_size, long long pages, const void* pool, const char* what) {
  // slots are 32-bit numbers; a slot's tile times the tiles of a page stays below 2^32 (see per_magic)
  if (hk > 0 && pages * page_size <= 0x7fffffffll && pages * page_size / kTile * (page_size / kTile) < (1ll << 32) && (d == 64 || d == 128 || d == 256) && page_size > 0 && page_size % kTile == 0 && (uintptr_t)pool % 16 == 0) return true;
  msgl_set_error_text(what);
  return false;
}

uint32_t magic(int per) { return (uint32_t)(((1ull << 32) + per - 1) / per); }
// four where threads of one row each would fill the GPU (2048 threads an SM) more than twice over
int rows_of_a_thread(long long rows, int hk, int d) { return rows * hk * (d / 8) > 2ll * 2048 * device_sms() ? 4 : 1; }

}  // namespace

MSGL_API int msgl_store_fp4(const void* k, const void* v, long long ldk, long long ldv, void* pool, const void* loc, const void* k_head,
                            const void* v_head, void* weights, int rows, int hk, int d, int page_size, long long pages, int dtype,
                            cudaStream_t stream) {
  if (rows <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pages, pool, "store_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens, fewer than 2^31 slots"))
    return MSGL_BAD_ARG;
  if (ldk % 8 || ldv % 8 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("store_kv_fp4: 16-bit rows on 16-byte boundaries");
    return MSGL_BAD_ARG;
  }
  RowArgs a{k, v, ldk, ldv, (uint8_t*)pool, 0, (const int32_t*)loc, (const float*)k_head, (const float*)v_head, (float*)weights,
            rows, hk, page_size / kTile, magic(page_size / kTile), pages * page_size};
  const int u = rows_of_a_thread(rows, hk, d);
  const long long threads = (long long)((rows + u - 1) / u) * hk * (d / 8);
  if (threads > 0x7fffff00ll) {
    msgl_set_error_text("store_kv_fp4: more rows than a launch has threads for");
    return MSGL_BAD_ARG;
  }
  const dim3 grid((unsigned)((threads + 255) / 256));
#define STORE(T, D, U) msgl_launch(store_fp4_kernel<T, D, U>, grid, dim3(256), 0, stream, a)
#define STORES(T, D) do { if (u == 1) STORE(T, D, 1); else STORE(T, D, 4); } while (0)
  if (dtype == MSGL_BF16) { if (d == 64) STORES(__nv_bfloat16, 64); else if (d == 128) STORES(__nv_bfloat16, 128); else STORES(__nv_bfloat16, 256); }
  else { if (d == 64) STORES(__half, 64); else if (d == 128) STORES(__half, 128); else STORES(__half, 256); }
#undef STORES
#undef STORE
  MSGL_CHECK_LAUNCH("store_kv_fp4");
  return MSGL_OK;
}

MSGL_API int msgl_load_fp4(const void* pool, long long layer_bytes, int layers, const void* loc, const void* k_head, const void* v_head,
                           void* k, void* v, int rows, int hk, int d, int page_size, long long pages, int dtype, cudaStream_t stream) {
  if (rows <= 0 || layers <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pages, pool, "load_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens, fewer than 2^31 slots"))
    return MSGL_BAD_ARG;
  if (dtype != MSGL_BF16 && dtype != MSGL_F16) {
    msgl_set_error_text("load_kv_fp4: rows of 16 bits");
    return MSGL_BAD_ARG;
  }
  RowArgs a{k, v, 0, 0, (uint8_t*)const_cast<void*>(pool), layer_bytes, (const int32_t*)loc, (const float*)k_head,
            (const float*)v_head, nullptr, rows, hk, page_size / kTile, magic(page_size / kTile), pages * page_size};
  const int u = rows_of_a_thread((long long)rows * layers, hk, d);
  const long long threads = (long long)((rows + u - 1) / u) * hk * (d / 8);
  if (threads > 0x7fffff00ll || layers > 65535) {
    msgl_set_error_text("load_kv_fp4: more rows than a launch has threads for");
    return MSGL_BAD_ARG;
  }
  const dim3 grid((unsigned)((threads + 255) / 256), layers);
#define LOAD(T, D, U) msgl_launch(load_fp4_kernel<T, D, U>, grid, dim3(256), 0, stream, a)
#define LOADS(T, D) do { if (u == 1) LOAD(T, D, 1); else LOAD(T, D, 4); } while (0)
  if (dtype == MSGL_BF16) { if (d == 64) LOADS(__nv_bfloat16, 64); else if (d == 128) LOADS(__nv_bfloat16, 128); else LOADS(__nv_bfloat16, 256); }
  else { if (d == 64) LOADS(__half, 64); else if (d == 128) LOADS(__half, 128); else LOADS(__half, 256); }
#undef LOADS
#undef LOAD
  MSGL_CHECK_LAUNCH("load_kv_fp4");
  return MSGL_OK;
}

MSGL_API int msgl_evict_fp4(void* pool, long long layer_bytes, void* weights, long long layer_weights, int layers, const void* table,
                            int width, const void* new_table, int new_width, const void* lens, void* kept, void* new_lens,
                            int requests, int hk, int d, int page_size, int pages, int budget, int recent, int sinks,
                            int max_kv, cudaStream_t stream) {
  if (requests <= 0 || layers <= 0) return MSGL_OK;
  if (!shape_ok(hk, d, page_size, pages, pool, "evict_kv_fp4: heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens, fewer than 2^31 slots"))
    return MSGL_BAD_ARG;
  if (budget <= 0 || recent < 0 || sinks < 0 || recent + sinks > budget || width <= 0 ||
      (long long)new_width * page_size < budget) {
    msgl_set_error_text("evict_kv_fp4: recent + sinks <= budget, and new pages for the budget");
    return MSGL_BAD_ARG;
  }
  EvictArgs a{(uint8_t*)pool, layer_bytes, (float*)weights, layer_weights, (const int32_t*)table, (const int32_t*)new_table,
              (int32_t*)kept, (int32_t*)new_lens, (const int32_t*)lens, width, new_width, requests, hk, page_size, pages, budget,
              recent, sinks, page_size / kTile, 0};
  a.per_magic = magic(a.per);
  a.wide = (uintptr_t)weights % 16 == 0 && layer_weights % 4 == 0;
  a.layers = layers;
  const long long units = (long long)layers * requests * hk, room = (long long)width * page_size;
  // i / 16 / per by a multiplication is exact while i / 16 times (per_magic * per - 2^32 < per) stays below 2^32
  if (room / kTile * a.per >= (1ll << 32) || room > 0x7fff0000ll || units > 0x7fffffffll) {
    msgl_set_error_text("evict_kv_fp4: a block table of fewer tokens");
    return MSGL_BAD_ARG;
  }
  a.by_length = requests > 1 && requests <= 32 && units > device_sms();
  const long long longest = max_kv > 0 && max_kv < room ? max_kv : room;
  if (longest <= kKeysInShared) {
    static bool ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeysInShared * 4);
      if (e != cudaSuccess) { msgl_set_error("evict_kv_fp4 shared memory", e); return MSGL_CUDA_ERROR; }
      if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    msgl_launch(evict_select_kernel<true>, dim3((unsigned)units), dim3(kSelThreads), (size_t)((longest + 3) / 4 * 16), stream, a, (int)longest);
  } else {
    msgl_launch(evict_select_kernel<false>, dim3((unsigned)units), dim3(kSelThreads), 0, stream, a, 0);
  }
  MSGL_CHECK_LAUNCH("evict_select");
  const int tiles = (budget + kTile - 1) / kTile;
  const dim3 grid((unsigned)((units * tiles + 7) / 8));
#define MOVE(D) msgl_launch(evict_move_kernel<D>, grid, dim3(256), 0, stream, a, tiles, units* tiles)
  if (d == 64) MOVE(64); else if (d == 128) MOVE(128); else MOVE(256);
#undef MOVE
  MSGL_CHECK_LAUNCH("evict_move");
  return MSGL_OK;
}
