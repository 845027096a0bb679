// Causal attention over the paged K/V pool of 4 bits (kv_fp4.cuh).
//
// A unit is a tile of rows of one request and key head, a row being a (query position, head of the group) pair, with all 16-token
// tiles that its request's rows see. The tiles of all units in a line are dealt evenly to the warps of the GPU; a warp
// fetches its tiles into a ring of its own (bulk copies of 18 D bytes) and keeps the softmax of the unit it is in. Units that a
// warp has whole are written at once, parts of others go to the workspace and a second kernel joins them.
//
// Both products take the cache as their first operand (rows: 16 tokens, or 16 channels), so a row tile is 8 queries wide and
// no product is spent on more rows than a group of 8 heads has: S^T = K Q^T, O^T = V^T P^T. Codes go e2m1 -> f16 (one
// conversion for two) and are multiplied by their scale, which is exact (2 + 4 significant bits). Queries are scaled to
// powers of two around 2^10 and taken as f16: exact for bf16 and fp16 values down to 2^-24 of a row's largest. Sums, running
// maximum and sum of the softmax are fp32. Probabilities go into the second product as f16 (11 bits) after a factor of 2^7,
// so that they are normal numbers down to 2^-21 of the largest; the maximum moves only when a score passes it by 2^8, which
// the factor leaves room for (2^15).
#include "kv_fp4.cuh"
#include "ptx.cuh"

using namespace msgl;
using namespace msgl::fp4;
using namespace msgl::ptx;

namespace {

constexpr int kWarps = 4;            // of a CTA
constexpr int kMost = 1024;          // requests of a launch
constexpr int kFewTiles = 4;         // a warp gets at least so many tiles
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kUp = 7.f, kSlack = 8.f;   // log2 of the probabilities' factor; by how much a score may pass the maximum

__device__ int g_fp4_status = 0;

struct Fp4Args {
  const void* q;
  void* out;
  const uint8_t* pool;
  const int32_t* table;
  long long table_stride;
  const int32_t* cu_q;
  const int32_t* lens;
  const float* k_head;
  const float* v_head;
  float* lse;               // [rows, hq], log2; null without weights
  float* weights;
  float* parts;             // [2 * workers][rows of a tile][D + 2]
  long long* line;          // [B + 2]: first tile of every request in the line, total; workers
  int width, B, hq, hk, group, page_size, per, pages, window, row_tile, workers;   // per: tiles of a page
  float scale;
  int* status;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// four bytes of two codes each -> four pairs of f16
__device__ __forceinline__ void widen(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// token of a tile in row g + 8 r of the keys' operand
__device__ __forceinline__ int token_of(int g, int r) { return 4 * (g >> 1) + 2 * r + (g & 1); }

// ---- the line of tiles -----------------------------------------------------------------
struct Request {
  int q0, q_len, n;         // first row, rows, tokens
  int tile0, tiles;         // tiles that its rows see
  int row_tiles;
  __device__ __forceinline__ void load(const Fp4Args& a, int b) {
    q0 = a.cu_q[b];
    q_len = a.cu_q[b + 1] - q0;
    n = min(max(a.lens[b], 0), a.width * a.page_size);
    const int lo = a.window > 0 ? max(0, n - q_len - a.window + 1) : 0;
    tile0 = lo / kTile;
    tiles = q_len > 0 && n > lo ? (n + kTile - 1) / kTile - tile0 : 0;
    row_tiles = (max(q_len, 0) * a.group + a.row_tile - 1) / a.row_tile;
  }
  __device__ __forceinline__ long long cost(const Fp4Args& a, bool whole_rows) const {
    return (long long)tiles * a.hk * (whole_rows ? 1 : row_tiles);
  }
};

// First tile of every request in `line` (kMost + 1 entries), the total in line[B].
__device__ __forceinline__ void lay_line(const Fp4Args& a, long long* line, bool whole_rows) {
  __shared__ long long sums[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.B + kWarps * 32 - 1) / (kWarps * 32);
  const int b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    Request r;
    r.load(a, b);
    line[b] = mine;
    mine += r.cost(a, whole_rows);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  long long before = incl - mine;
  for (int w = 0; w < warp; ++w) before += sums[w];
  for (int b = b0; b < b1; ++b) line[b] += before;
  if (threadIdx.x == kWarps * 32 - 1) line[a.B] = before + mine;
  __syncthreads();
}

// Worker w of W has tiles [begin(w), begin(w + 1)).
struct Deal {
  long long base;
  int workers, extra;
  __device__ __forceinline__ Deal(long long total, int most) {
    workers = (int)max(1ll, min((long long)most, total / kFewTiles));
    base = total / workers;
    extra = (int)(total - base * workers);
  }
  __device__ __forceinline__ long long begin(int w) const { return w * base + min(w, extra); }
  __device__ __forceinline__ int owner(long long at) const {
    const long long big = (base + 1) * extra;
    return (int)(at < big ? at / (base + 1) : extra + (at - big) / max(base, 1ll));
  }
};

// A place in the line: a row tile (rt) of a key head of request b, and a tile of 16 tokens: sub of the page in column col of
// the block table. Steps take no divisions.
struct Walk {
  int b, head, rt, tile, col, sub;
  Request r;
  __device__ __forceinline__ void start_unit(const Fp4Args& a) {
    tile = 0;
    col = r.tile0 / a.per;
    sub = r.tile0 - col * a.per;
  }
  __device__ __forceinline__ void seek(const Fp4Args& a, const long long* line, long long at, bool whole_rows) {
    int lo = 0, hi = a.B - 1;                   // the last request that starts at or before `at` has it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (line[mid] <= at) lo = mid; else hi = mid - 1;
    }
    b = lo;
    r.load(a, b);
    const long long o = at - line[b];
    const int unit = (int)(o / max(r.tiles, 1)), row_tiles = whole_rows ? 1 : max(r.row_tiles, 1);
    tile = (int)(o - (long long)unit * r.tiles);
    head = unit / row_tiles;
    rt = unit - head * row_tiles;
    col = (r.tile0 + tile) / a.per;
    sub = r.tile0 + tile - col * a.per;
  }
  // on to the next unit that has tiles
  __device__ __forceinline__ void next_unit(const Fp4Args& a, const long long* line, bool whole_rows) {
    if (!whole_rows && ++rt < r.row_tiles) { start_unit(a); return; }
    rt = 0;
    if (++head == a.hk) {
      head = 0;
      do ++b; while (b < a.B - 1 && line[b] == line[b + 1]);
      r.load(a, min(b, a.B - 1));
    }
    start_unit(a);
  }
  // true where another unit begins
  __device__ __forceinline__ bool next(const Fp4Args& a, const long long* line, bool whole_rows) {
    if (++sub == a.per) { sub = 0; ++col; }
    if (++tile < r.tiles) return false;
    next_unit(a, line, whole_rows);
    return true;
  }
  __device__ __forceinline__ int page(const Fp4Args& a) const {
    const int page = a.table[(long long)b * a.table_stride + col];
    (void)MSGL_OOB(page, a.pages);
    return min(max(page, 0), a.pages - 1);
  }
  template <int D> __device__ __forceinline__ const uint8_t* address(const Fp4Args& a, int page) const {
    return a.pool + (long long)((page * a.hk + head) * a.per + sub) * Tile<D>::bytes;
  }
};

// ---- queries ---------------------------------------------------------------------------
// Lane 4 g + j takes channels j D / 4 .. of row g as the second operand of S^T, scaled by a power of two; returns what the
// row's scores have to be multiplied by.
template <typename T, int D>
__device__ __forceinline__ float load_query(const Fp4Args& a, const Request& r, int head, int row, int lane, uint32_t (&qf)[D / 8]) {
  const bool there = row < r.q_len * a.group;
  const int pos = there ? row / a.group : 0;
  const T* src = reinterpret_cast<const T*>(a.q) + ((long long)(r.q0 + pos) * a.hq + head * a.group + (there ? row - pos * a.group : 0)) * D
                 + (lane & 3) * (D / 4);
  float top = 0.f;
  Vec8<T> raw[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    if (there) raw[i] = *reinterpret_cast<const Vec8<T>*>(src + 8 * i);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[i].v[e] = Pack2<T>::make(0.f, 0.f);
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int ex = (int)(__float_as_uint(top) >> 23);            // 0: zeros; 255: infinite
  const int up = top > 0.f && ex < 255 ? min(max(137 - ex, -126), 126) : 0;
  const float f = copysignf(__uint_as_float((uint32_t)(127 + up) << 23), a.scale);     // a negative scale: on the query
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 4; ++e) qf[4 * i + e] = f16x2(x[2 * e] * f, x[2 * e + 1] * f);
  }
  return __uint_as_float((uint32_t)(127 - up) << 23);
}

template <int D> struct Raw {          // a lane's share of a tile
  uint4 k[D / 64], v[D / 64];
  uint32_t ks[D / 128 > 0 ? D / 128 : 1], vs[D / 128 > 0 ? D / 128 : 1];
};

template <int D> __device__ __forceinline__ void load_keys(const uint8_t* tile, int lane, Raw<D>& x) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) x.k[i] = *reinterpret_cast<const uint4*>(tile + 512 * i + 16 * lane);
  if (D == 64) x.ks[0] = *reinterpret_cast<const uint16_t*>(tile + Tile<D>::k_sf + 2 * lane);
  else
#pragma unroll
    for (int i = 0; i < D / 128; ++i) x.ks[i] = *reinterpret_cast<const uint32_t*>(tile + Tile<D>::k_sf + lane * (D / 32) + 4 * i);
}
template <int D> __device__ __forceinline__ void load_values(const uint8_t* tile, int lane, Raw<D>& x) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) x.v[i] = *reinterpret_cast<const uint4*>(tile + Tile<D>::v + 512 * i + 16 * lane);
  const int g = lane >> 2, j = lane & 3;
#pragma unroll
  for (int i = 0; i < (D == 256 ? 2 : 1); ++i) {
    const int block = D == 64 ? g >> 1 : D == 128 ? g : 2 * g + i;
    x.vs[i] = *reinterpret_cast<const uint32_t*>(tile + Tile<D>::v_sf + (block * 4 + j) * 4);
  }
}
__device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Keys of row r, block of 32 bits w (8 channels): D / 32 words of each row.
template <int D> __device__ __forceinline__ uint32_t key_word(const Raw<D>& x, int r, int w) {
  const int at = r * (D / 32) + w;
  return word(x.k[at / 4], at % 4);
}
// scale of row r, block i (of D / 64), in both halves
template <int D> __device__ __forceinline__ uint32_t key_scale(const Raw<D>& x, int r, int i) {
  const int at = r * (D / 64) + i;                                  // byte
  const uint32_t two = widen_e4m3(x.ks[at / 4] >> (at % 4 / 2 * 16));
  return __byte_perm(two, two, at % 2 ? 0x3232 : 0x1010);
}

// S^T of the tile for NB blocks of 8 rows
template <int D, int NB> __device__ __forceinline__ void scores(const Raw<D>& x, const uint32_t (&qf)[NB][D / 8], float (&s)[NB][4]) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {                                // blocks of 16 channels: 2 words, 4 products
    const uint32_t s0 = key_scale<D>(x, 0, i), s1 = key_scale<D>(x, 1, i);
#pragma unroll
    for (int w = 2 * i; w < 2 * i + 2; ++w) {
      uint32_t h0[4], h1[4];
      widen(key_word<D>(x, 0, w), h0);
      widen(key_word<D>(x, 1, w), h1);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t a0 = times(h0[2 * c], s0), a1 = times(h1[2 * c], s1), a2 = times(h0[2 * c + 1], s0), a3 = times(h1[2 * c + 1], s1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma(s[nb], a0, a1, a2, a3, qf[nb][4 * w + 2 * c], qf[nb][4 * w + 2 * c + 1]);
      }
    }
  }
}

// CTAs on an SM: what the registers allow without spilling the loop's values
__host__ __device__ constexpr int ctas_of(int d, int nb) { return d == 256 ? (nb == 1 ? 3 : 2) : nb == 1 ? (d == 64 ? 5 : 4) : nb == 2 ? 3 : 2; }

template <int D, int NB> struct Shape {
  static constexpr int stages = D == 64 ? 4 : 2;         // of two tiles
  static constexpr int ring = kWarps * stages * 2 * Tile<D>::bytes;
  static constexpr int ctas = ctas_of(D, NB);
  static constexpr int smem = ring + kWarps * stages * 8 + 16 + (kMost + 2) * 8;
};

template <typename T, int D, int NB>
__global__ void __launch_bounds__(kWarps * 32, Shape<D, NB>::ctas) fp4_attention_kernel(const Fp4Args a) {
  constexpr int STAGES = Shape<D, NB>::stages, BYTES = Tile<D>::bytes;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + warp * STAGES * 2 * BYTES;
  const uint32_t bar = smem_u32(smem + Shape<D, NB>::ring) + warp * STAGES * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Shape<D, NB>::ring + kWarps * STAGES * 8);
  long long* line = reinterpret_cast<long long*>(smem + Shape<D, NB>::ring + kWarps * STAGES * 8 + 16);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bar + 8 * s, 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_enter();
  lay_line(a, line, false);
  const Deal deal(line[a.B], a.workers);
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= a.B; b += kWarps * 32) a.line[b] = line[b];
  }
  // neighbours in the line lie on different SMs: a short line is spread over all of them
  const int worker = warp * gridDim.x + blockIdx.x;
  if (worker >= deal.workers) return;
  const long long at = deal.begin(worker);
  const int total = (int)(deal.begin(worker + 1) - at);     // tiles
  if (total <= 0) return;

  // Tiles come in pairs, a stage for each. Lane i finds the places of pairs i, 32 + i, ... and fetches them: no step along the
  // line for each tile.
  const int pairs = (total + 1) / 2;
  const uint8_t *mine0 = nullptr, *mine1 = nullptr;
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched % 32 == 0) {
      Walk w;
      w.seek(a, line, at + min(2 * (fetched + lane), total - 1), false);
      mine0 = w.address<D>(a, w.page(a));
      w.seek(a, line, at + min(2 * (fetched + lane) + 1, total - 1), false);
      mine1 = w.address<D>(a, w.page(a));
    }
    if (lane == fetched % 32) {
      const bool both = 2 * fetched + 1 < total;
      const uint32_t full = bar + 8 * stage, to = smem_u32(ring + stage * 2 * BYTES);
      mbar_expect_tx(full, both ? 2 * BYTES : BYTES);
      bulk_load(to, mine0, BYTES, full);
      if (both) bulk_load(to + BYTES, mine1, BYTES, full);
    }
    ++fetched;
  };
  for (int s = 0; s < STAGES && s < pairs; ++s) fetch(s);
  Walk get;
  get.seek(a, line, at, false);

  const int g = lane >> 2, j = lane & 3;
  int done = 0, stage = 0;       // done: tiles; stage: of the next one
  uint32_t phase = 0;
  bool ok = true;
  while (done < total) {
    // ---- one unit, or this warp's part of it
    const int first = get.tile, head = get.head, row0 = get.rt * a.row_tile;
    const int count = min(total - done, get.r.tiles - first);
    const Request r = get.r;
    const int rows = min(a.row_tile, r.q_len * a.group - row0);
    uint32_t qf[NB][D / 8];
    float c[NB][2];              // factors of the scores of rows 2 j and 2 j + 1, above 0
    const float kh = fabsf(a.scale) * kLog2e * (a.k_head != nullptr ? a.k_head[head] : 1.f);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float back = load_query<T, D>(a, r, head, row0 + nb * 8 + g, lane, qf[nb]);
      c[nb][0] = fmaxf(kh * __shfl_sync(0xffffffffu, back, 8 * j), 1e-37f);
      c[nb][1] = fmaxf(kh * __shfl_sync(0xffffffffu, back, 8 * j + 4), 1e-37f);
    }
    // m: running maxima; base: what is taken from a score in the exponent
    float o[NB][D / 16][4], m[NB][2], base[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
      m[nb][0] = m[nb][1] = -INFINITY;
      base[nb][0] = base[nb][1] = -kUp;
      l[nb][0] = l[nb][1] = 0.f;
    }
    // tokens [lo_all, hi_all) are seen by all rows
    const int pos0 = r.n - r.q_len + row0 / a.group, pos1 = r.n - r.q_len + (row0 + rows - 1) / a.group;
    const int hi_all = pos0 + 1, lo_all = a.window > 0 ? pos1 - a.window + 1 : 0;

    for (int t = 0; t < count;) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar + 8 * stage, phase, abort_flag, a.status, 401));
      if (!ok) break;
      const uint8_t* tile = ring + stage * 2 * BYTES;
      // of the stage's tiles one may be another unit's: `from` .. `to` are the tokens of this one, tok0 is the stage's first
      const int u0 = done & 1, from = u0 * kTile, to = min(2, u0 + count - t) * kTile;
      const int tok0 = (r.tile0 + first + t - u0) * kTile;
      if (tok0 + from <= pos1) {                               // else rows behind these see it
        float s[2][NB][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Raw<D> x;
          load_keys<D>(tile + u * BYTES, lane, x);
          scores<D, NB>(x, qf, s[u]);
        }
        const bool ragged = tok0 + 2 * kTile > hi_all || tok0 < lo_all || to - from < 2 * kTile;
        bool move = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (ragged) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int pos = r.n - r.q_len + (row0 + nb * 8 + 2 * j + k) / a.group;
              const int hi = min(min(pos + 1, r.n) - tok0, to), lo = max(a.window > 0 ? pos - a.window + 1 - tok0 : 0, from);
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int tok = u * kTile + token_of(g, h);
                  if (tok >= hi || tok < lo) s[u][nb][2 * h + k] = -INFINITY;
                }
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
            move |= fmaxf(fmaxf(s[0][nb][k], s[0][nb][2 + k]), fmaxf(s[1][nb][k], s[1][nb][2 + k])) * c[nb][k] > m[nb][k] + kSlack;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float top = fmaxf(fmaxf(s[0][nb][k], s[0][nb][2 + k]), fmaxf(s[1][nb][k], s[1][nb][2 + k])) * c[nb][k];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              top = fmaxf(top, m[nb][k]);
              const float f = m[nb][k] == top ? 1.f : exp2_fast(m[nb][k] - top);
              m[nb][k] = top;
              base[nb][k] = (top == -INFINITY ? 0.f : top) - kUp;
              l[nb][k] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[nb][i][k] *= f; o[nb][i][2 + k] *= f; }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t p0[NB], p1[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float e0 = exp2_fast(fmaf(s[u][nb][0], c[nb][0], -base[nb][0])), e1 = exp2_fast(fmaf(s[u][nb][1], c[nb][1], -base[nb][1])),
                        e2 = exp2_fast(fmaf(s[u][nb][2], c[nb][0], -base[nb][0])), e3 = exp2_fast(fmaf(s[u][nb][3], c[nb][1], -base[nb][1]));
            l[nb][0] += e0 + e2;
            l[nb][1] += e1 + e3;
            p0[nb] = transpose8(f16x2(e0, e1));
            p1[nb] = transpose8(f16x2(e2, e3));
          }
          Raw<D> x;
          load_values<D>(tile + u * BYTES, lane, x);
          // values of tokens that no row sees may be anything; a NaN that only some rows see must not reach the others
          uint32_t nan_mask = 0;       // bit 4 i + e: token 4 j + e has no number in block i of the lane's channels
          if (ragged) {
#pragma unroll
            for (int i = 0; i < (D == 256 ? 2 : 1); ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((x.vs[i] >> (8 * e) & 0x7F) == 0x7F) {
                  nan_mask |= 1u << (4 * i + e);
                  x.vs[i] &= ~(0xFFu << (8 * e));
                }
          }
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {                  // words of 8 channels of the lane: 4 products
            const int i = D == 256 ? w / 2 : 0;
            const uint32_t s01 = widen_e4m3(x.vs[i]), s23 = widen_e4m3(x.vs[i] >> 16);
            uint32_t tw[4];                                    // of tokens 4 j .. 4 j + 3
#pragma unroll
            for (int e = 0; e < 4; ++e) { const int k = e * (D / 64) + w; tw[e] = word(x.v[k / 4], k % 4); }
            uint32_t lo01[4], hi01[4], lo23[4], hi23[4];       // pairs of tokens of the even and of the odd channels
            widen((tw[0] & 0x0F0F0F0Fu) | ((tw[1] << 4) & 0xF0F0F0F0u), lo01);
            widen(((tw[0] >> 4) & 0x0F0F0F0Fu) | (tw[1] & 0xF0F0F0F0u), hi01);
            widen((tw[2] & 0x0F0F0F0Fu) | ((tw[3] << 4) & 0xF0F0F0F0u), lo23);
            widen(((tw[2] >> 4) & 0x0F0F0F0Fu) | (tw[3] & 0xF0F0F0F0u), hi23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a0 = times(lo01[k], s01), a1 = times(hi01[k], s01), a2 = times(lo23[k], s23), a3 = times(hi23[k], s23);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) mma(o[nb][4 * w + k], a0, a1, a2, a3, p0[nb], p1[nb]);
            }
          }
          if (ragged && __any_sync(0xffffffffu, nan_mask != 0)) {
            for (int jj = 0; jj < 4; ++jj) {
              const uint32_t bits = __shfl_sync(0xffffffffu, nan_mask, 4 * g + jj);
              for (int e = 0; e < 4; ++e) {
                const int tok = u * kTile + 4 * jj + e;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int c = 0; c < 2; ++c) {
                    const int pos = r.n - r.q_len + (row0 + nb * 8 + 2 * j + c) / a.group;
                    const bool seen = tok < min(min(pos + 1, r.n) - tok0, to) && tok >= from &&
                                      !(a.window > 0 && tok0 + tok <= pos - a.window);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                      if (seen && (bits >> ((D == 256 ? i / 8 * 4 : 0) + e) & 1)) o[nb][i][c] = o[nb][i][2 + c] = NAN;
                  }
              }
            }
          }
        }
      }
      t += (to - from) / kTile;
      done += (to - from) / kTile;
      if (to == 2 * kTile) {
        __syncwarp();
        if (fetched < pairs) fetch(stage);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) break;

    // ---- rows 2 j and 2 j + 1 of every block: channels g D / 8 .. (D / 8 of them)
    const bool whole = first == 0 && count == r.tiles;
    const float vh = a.v_head != nullptr ? a.v_head[head] : 1.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], d);
        const int row = nb * 8 + 2 * j + c;
        if (row >= rows) continue;
        if (whole) {
          const float f = l[nb][c] > 0.f || l[nb][c] != l[nb][c] ? vh / l[nb][c] : 0.f;
          const int qi = (row0 + row) / a.group;
          const long long to = (long long)(r.q0 + qi) * a.hq + head * a.group + (row0 + row - qi * a.group);
          T* dst = reinterpret_cast<T*>(a.out) + to * D + g * (D / 8);
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) { y[2 * e] = o[nb][4 * i + e][c] * f; y[2 * e + 1] = o[nb][4 * i + e][2 + c] * f; }
            store8(dst + 8 * i, y);
          }
          if (a.lse != nullptr && g == 0) a.lse[to] = (m[nb][c] == -INFINITY ? 0.f : m[nb][c]) - kUp + log2f(l[nb][c]);
        } else {
          float* part = a.parts + ((long long)(2 * worker + (first == 0 ? 1 : 0)) * a.row_tile + row) * (D + 4);
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) { y[2 * e] = o[nb][4 * i + e][c]; y[2 * e + 1] = o[nb][4 * i + e][2 + c]; }
            store8(part + g * (D / 8) + 8 * i, y);
          }
          if (g == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m[nb][c], l[nb][c]);
        }
      }
    }
    if (done < total) get.next_unit(a, line, false);
  }
  if (!ok) {     // copies may be in flight: they land before the shared memory goes
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

// Rows of units that several workers share, or that see nothing: the parts joined. SPREAD warps of a CTA take the parts of one
// (row, query head) in turn.
template <typename T, int D, int SPREAD> __global__ void __launch_bounds__(256) fp4_join_kernel(const Fp4Args a, int total_rows) {
  constexpr int E = D / 32, AHEAD = 4;
  __shared__ float sum[8][D + 2];
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long id = (long long)blockIdx.x * (8 / SPREAD) + warp / SPREAD;
  const int row = (int)(id / a.hq), qh = (int)(id - (long long)row * a.hq), mine = warp % SPREAD;
  // of another launch, or of no request; the CTA's rows may differ in it
  bool there = id < (long long)total_rows * a.hq && row >= a.cu_q[0] && row < a.cu_q[a.B], empty = false;
  float m = -INFINITY, l = 0.f, y[E] = {};
  int head = 0;
  if (there) {
    int lo = 0, hi = a.B - 1;                             // the last request that starts at or before the row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    Request r;
    r.load(a, lo);
    empty = r.tiles == 0;
    if (!empty) {
      const Deal deal(a.line[a.B], a.workers);
      head = qh / a.group;
      const int in_unit = (row - r.q0) * a.group + qh - head * a.group;
      const int rt = in_unit / a.row_tile, in_tile = in_unit - rt * a.row_tile;
      const long long u0 = a.line[lo] + ((long long)head * r.row_tiles + rt) * r.tiles;
      const int w0 = deal.owner(u0), w1 = deal.owner(u0 + r.tiles - 1);
      there = w0 != w1;                                   // else written by its worker
      for (int wb = w0 + mine; there && wb <= w1; wb += AHEAD * SPREAD) {
        float2 ml[AHEAD];
        float x[AHEAD][E];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int w = wb + i * SPREAD;
          ml[i] = make_float2(-INFINITY, 0.f);
          const float* part = a.parts + ((long long)(2 * w + (w == w0 ? 1 : 0)) * a.row_tile + in_tile) * (D + 4);
          if (w <= w1) ml[i] = *reinterpret_cast<const float2*>(part + D);
#pragma unroll
          for (int e = 0; e < E; ++e) x[i][e] = w <= w1 ? part[lane * E + e] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const float top = fmaxf(m, ml[i].x);
          const float f0 = m == top ? 1.f : exp2_fast(m - top), f1 = ml[i].x == top ? 1.f : exp2_fast(ml[i].x - top);
          m = top;
          l = l * f0 + ml[i].y * f1;
#pragma unroll
          for (int e = 0; e < E; ++e) y[e] = y[e] * f0 + x[i][e] * f1;
        }
      }
    }
  }
  if (SPREAD > 1) {
    if (mine != 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) sum[warp][lane * E + e] = y[e];
      if (lane == 0) { sum[warp][D] = m; sum[warp][D + 1] = l; }
    }
    __syncthreads();
    if (mine != 0) return;
    for (int k = 1; k < SPREAD; ++k) {
      const float* o = sum[warp + k];
      const float top = fmaxf(m, o[D]), f0 = m == top ? 1.f : exp2_fast(m - top), f1 = o[D] == top ? 1.f : exp2_fast(o[D] - top);
      m = top;
      l = l * f0 + o[D + 1] * f1;
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = y[e] * f0 + o[lane * E + e] * f1;
    }
  }
  if (!there) return;
  const float f = l > 0.f || l != l ? (a.v_head != nullptr ? a.v_head[head] : 1.f) / l : 0.f;
  if (a.lse != nullptr && lane == 0 && !empty) a.lse[id] = (m == -INFINITY ? 0.f : m) - kUp + log2f(l);
  T* dst = reinterpret_cast<T*>(a.out) + id * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<typename Pack2<T>::type*>(dst + e) = Pack2<T>::make(y[e] * f, y[e + 1] * f);
}

// What the rows give every token: the keys once more, with the rows' final maxima and sums. A tile's keys go through all rows of
// their (request, key head) pair, so a token's sum is taken by one lane in one order. MANY false: up to 8 rows, in registers;
// warps deal out the tiles of all pairs. MANY: CTAs do; the pair's queries lie in shared memory, kChunk blocks of 8 rows at
// a time, and the warps take the CTA's tiles in turn. A warp has four tiles' keys under way.
template <int D, bool MANY> struct WeightsShape {
  static constexpr int stages = 4, key_bytes = 9 * D;                  // codes and scales
  static constexpr int chunk = !MANY ? 0 : D == 256 ? 4 : 8;           // blocks of 8 rows
  static constexpr int ctas = D == 256 ? 2 : 4;
  static constexpr int ring = kWarps * stages * key_bytes, bars = ring, slots = bars + kWarps * stages * 8;
  static constexpr int flag = slots + kWarps * stages * 4, line = flag + 16, queries = line + (kMost + 2) * 8;
  static constexpr int rows = queries + chunk * 16 * D, smem = rows + chunk * 8 * 8;
};

// keys of a tile as the first operand
template <int D> __device__ __forceinline__ void key_operand(const Raw<D>& x, uint32_t (&k)[D / 16][4]) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint32_t s0 = key_scale<D>(x, 0, i), s1 = key_scale<D>(x, 1, i);
#pragma unroll
    for (int w = 2 * i; w < 2 * i + 2; ++w) {
      uint32_t h0[4], h1[4];
      widen(key_word<D>(x, 0, w), h0);
      widen(key_word<D>(x, 1, w), h1);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        k[2 * w + c][0] = times(h0[2 * c], s0);
        k[2 * w + c][1] = times(h1[2 * c], s1);
        k[2 * w + c][2] = times(h0[2 * c + 1], s0);
        k[2 * w + c][3] = times(h1[2 * c + 1], s1);
      }
    }
  }
}

template <typename T, int D, bool MANY>
__global__ void __launch_bounds__(kWarps * 32, WeightsShape<D, MANY>::ctas) fp4_weights_kernel(const Fp4Args a) {
  using S = WeightsShape<D, MANY>;
  constexpr int STAGES = S::stages;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  uint8_t* ring = smem + warp * STAGES * S::key_bytes;
  const uint32_t bar = smem_u32(smem + S::bars) + warp * STAGES * 8;
  int* slots = reinterpret_cast<int*>(smem + S::slots) + warp * STAGES;        // of the pool: the stages' tiles
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::flag);
  long long* line = reinterpret_cast<long long*>(smem + S::line);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bar + 8 * s, 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_enter();
  lay_line(a, line, true);
  const Deal deal(line[a.B], MANY ? gridDim.x : gridDim.x * kWarps);
  const int worker = MANY ? blockIdx.x : warp * gridDim.x + blockIdx.x;
  if (worker >= deal.workers) return;
  long long at = deal.begin(worker);
  const long long end = deal.begin(worker + 1);
  if (at >= end) return;

  // tiles first, first + step, ... of the line, `count` of them
  long long first = at;
  const int step = MANY ? kWarps : 1;
  int count = 0, fetched = 0, done = 0, uses = 0, mine = 0;        // uses: stages used up before this run of tiles
  auto fetch = [&]() {
    if (fetched % 32 == 0) {
      Walk w;
      w.seek(a, line, first + (long long)min(fetched + lane, count - 1) * step, true);
      mine = (w.page(a) * a.hk + w.head) * a.per + w.sub;
    }
    if (lane == fetched % 32) {
      const int s = (uses + fetched) % STAGES;
      const uint8_t* tile = a.pool + (long long)mine * Tile<D>::bytes;
      const uint32_t to = smem_u32(ring + s * S::key_bytes);
      slots[s] = mine;
      mbar_expect_tx(bar + 8 * s, S::key_bytes);
      bulk_load(to, tile, 8 * D, bar + 8 * s);
      bulk_load(to + 8 * D, tile + Tile<D>::k_sf, D, bar + 8 * s);
    }
    ++fetched;
  };
  uint32_t k[D / 16][4];
  int slot = 0;
  bool ok = true;
  auto next_keys = [&]() {          // waits for the next tile, takes its keys and lets another one in
    const int s = (uses + done) % STAGES;
    ok = __all_sync(0xffffffffu, ok && mbar_wait(bar + 8 * s, (uses + done) / STAGES & 1, abort_flag, a.status, 402));
    if (!ok) return;
    Raw<D> x;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) x.k[i] = *reinterpret_cast<const uint4*>(ring + s * S::key_bytes + 512 * i + 16 * lane);
    const uint8_t* sf = ring + s * S::key_bytes + 8 * D + lane * (D / 32);
    if (D == 64) x.ks[0] = *reinterpret_cast<const uint16_t*>(sf);
    else
#pragma unroll
      for (int i = 0; i < D / 128; ++i) x.ks[i] = *reinterpret_cast<const uint32_t*>(sf + 4 * i);
    slot = slots[s];
    key_operand<D>(x, k);
    __syncwarp();
    ++done;
    if (fetched < count) fetch();
    __syncwarp();
  };
  // weights that the two rows 2 j, 2 j + 1 of a block give tokens of rows g and g + 8
  auto given = [&](const Request& r, int row0, int tok0, const float (&s)[4], float cA, float cB, float eA, float eB, float& s0, float& s1) {
    const int posA = r.n - r.q_len + (row0 + 2 * j) / a.group, posB = r.n - r.q_len + (row0 + 2 * j + 1) / a.group;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = tok0 + token_of(g, i >> 1), pos = i & 1 ? posB : posA;
      const float c = i & 1 ? cB : cA, e = i & 1 ? eB : eA;
      const bool seen = tok <= min(pos, r.n - 1) && !(a.window > 0 && tok <= pos - a.window);
      const float p = seen && e != INFINITY ? exp2_fast(s[i] * c - e) : 0.f;
      if (i < 2) s0 += p; else s1 += p;
    }
  };
  auto give = [&](const Request& r, int tok0, float s0, float s1) {
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, d);
      s1 += __shfl_xor_sync(0xffffffffu, s1, d);
    }
    const int t = token_of(g, j & 1);      // lane 0 of the four has row g's token, lane 1 row g + 8's
    if (j < 2 && tok0 + t < r.n) atomicAdd(a.weights + (long long)slot * kTile + t, j ? s1 : s0);
  };
  auto lse_of = [&](const Request& r, int head, int row) {
    if (row >= r.q_len * a.group) return INFINITY;         // weight 0
    const int qi = row / a.group;
    return a.lse[(long long)(r.q0 + qi) * a.hq + head * a.group + row - qi * a.group];
  };
  Walk get;
  get.seek(a, line, at, true);
  if constexpr (!MANY) {
    count = (int)(end - at);
    for (int s = 0; s < min(STAGES, count); ++s) fetch();
    __syncwarp();
    uint32_t qf[D / 8];
    float cA = 0.f, cB = 0.f, eA = 0.f, eB = 0.f;
    bool fresh = true;
    while (done < count) {
      if (fresh) {
        const float back = load_query<T, D>(a, get.r, get.head, g, lane, qf);
        const float kh = fabsf(a.scale) * kLog2e * (a.k_head != nullptr ? a.k_head[get.head] : 1.f);
        cA = kh * __shfl_sync(0xffffffffu, back, 8 * j);
        cB = kh * __shfl_sync(0xffffffffu, back, 8 * j + 4);
        eA = lse_of(get.r, get.head, 2 * j);
        eB = lse_of(get.r, get.head, 2 * j + 1);
      }
      next_keys();
      if (!ok) break;
      float s[4] = {};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) mma(s, k[i][0], k[i][1], k[i][2], k[i][3], qf[2 * i], qf[2 * i + 1]);
      const int tok0 = (get.r.tile0 + get.tile) * kTile;
      float s0 = 0.f, s1 = 0.f;
      given(get.r, 0, tok0, s, cA, cB, eA, eB, s0, s1);
      give(get.r, tok0, s0, s1);
      if (done < count) fresh = get.next(a, line, true);
    }
  } else {
    uint4* queries = reinterpret_cast<uint4*>(smem + S::queries);      // [block][D / 32 pieces of 16 bytes][lane]
    float2* rowc = reinterpret_cast<float2*>(smem + S::rows);          // factor and log of the sum of a row
    while (at < end) {
      const Request r = get.r;
      const int head = get.head, seg = (int)min(end - at, (long long)(r.tiles - get.tile)), rows = r.q_len * a.group;
      const float kh = fabsf(a.scale) * kLog2e * (a.k_head != nullptr ? a.k_head[head] : 1.f);
      for (int row0 = 0; row0 < rows; row0 += 8 * S::chunk) {
        __syncthreads();                                               // the last chunk has been used
        const int blocks = min(S::chunk, (rows - row0 + 7) / 8);
        for (int nb = warp; nb < blocks; nb += kWarps) {
          uint32_t qf[D / 8];
          const float back = load_query<T, D>(a, r, head, row0 + nb * 8 + g, lane, qf);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) queries[(nb * (D / 32) + i) * 32 + lane] = make_uint4(qf[4 * i], qf[4 * i + 1], qf[4 * i + 2], qf[4 * i + 3]);
          if (j == 0) rowc[nb * 8 + g] = make_float2(kh * back, lse_of(r, head, row0 + nb * 8 + g));
        }
        __syncthreads();
        uses += count;                                                 // (of the run before: all of its tiles were taken)
        first = at + warp;
        count = seg > warp ? (seg - warp + kWarps - 1) / kWarps : 0;
        fetched = done = 0;
        if (ok)
          for (int s = 0; s < min(STAGES, count); ++s) fetch();
        __syncwarp();
        while (done < count && ok) {
          const int tok0 = (r.tile0 + get.tile + warp + done * kWarps) * kTile;
          next_keys();
          if (!ok) break;
          float s0 = 0.f, s1 = 0.f;
          for (int nb = 0; nb < blocks; ++nb) {
            float s[4] = {};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const uint4 q = queries[(nb * (D / 32) + i) * 32 + lane];
              mma(s, k[2 * i][0], k[2 * i][1], k[2 * i][2], k[2 * i][3], q.x, q.y);
              mma(s, k[2 * i + 1][0], k[2 * i + 1][1], k[2 * i + 1][2], k[2 * i + 1][3], q.z, q.w);
            }
            const float4 c = *reinterpret_cast<const float4*>(rowc + nb * 8 + 2 * j);
            given(r, row0 + nb * 8, tok0, s, c.x, c.z, c.y, c.w, s0, s1);
          }
          give(r, tok0, s0, s1);
        }
      }
      at += seg;
      if (at < end) get.next_unit(a, line, true);
    }
  }
  if (!ok) {     // copies may be in flight: they land before the shared memory goes
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

// Rows that a prompt step sees, in 16 bits, for the tensor-core kernel of prompts (attention_tc.cu): keys [Hk][t_cap][128] and
// values transposed [Hk][128][t_cap], zeros where a request has no token and behind the 64 channels of narrow heads; the heads'
// factors go to scores and output there. A warp has a tile and a head: values leave 16 tokens of a channel at a time (32
// bytes), as the lanes hold them. Bound: the 512 bytes written for a token and head.
template <typename T, int D> __global__ void __launch_bounds__(256)
fp4_gather_kernel(const Fp4Args a, T* __restrict__ kc, T* __restrict__ vt, const int* __restrict__ blk_req, const int* __restrict__ req_info,
                  long long t_cap, int tiles) {
  pdl_enter();
  const int lane = threadIdx.x & 31, id = blockIdx.x * 8 + (threadIdx.x >> 5), g = lane >> 2, j = lane & 3;
  if (id >= tiles) return;
  const int h = blockIdx.y, t0 = id * kTile, req = blk_req[t0 >> 7];
  const int tok0 = t0 - req_info[3 * req] + req_info[3 * req + 2], n = req_info[3 * req + 1];
  Raw<D> x = {};
  if (tok0 < n) {
    int page = a.table[(long long)req * a.table_stride + min(tok0 / a.page_size, a.width - 1)];
    (void)MSGL_OOB(page, a.pages);
    page = min(max(page, 0), a.pages - 1);
    const uint8_t* tile = a.pool + ((long long)(page * a.hk + h) * a.per + tok0 / kTile % a.per) * Tile<D>::bytes;
    load_keys<D>(tile, lane, x);
    load_values<D>(tile, lane, x);
  }
  auto to_t = [](uint32_t f16) {
    if (sizeof(T) == 2 && __is_same(T, __half)) return f16;
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&b);
  };
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = token_of(g, r);
    const bool there = tok0 + t < n;
    T* row = kc + ((long long)h * t_cap + t0 + t) * 128;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      uint32_t k[4];
      widen(key_word<D>(x, r, w), k);
      const uint32_t s = key_scale<D>(x, r, w / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = there ? to_t(times(k[i], s)) : 0u;
      *reinterpret_cast<uint4*>(row + j * (D / 4) + 8 * w) = make_uint4(k[0], k[1], k[2], k[3]);
    }
    if (D == 64)
#pragma unroll
      for (int w = 0; w < 2; ++w) *reinterpret_cast<uint4*>(row + 64 + j * 16 + 8 * w) = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)                  // what lies behind the request may be anything
    if (tok0 + 4 * j + e >= n) x.vs[0] &= ~(0xFFu << (8 * e));
  const uint32_t s01 = widen_e4m3(x.vs[0]), s23 = widen_e4m3(x.vs[0] >> 16);
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
    uint32_t tw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { const int k = e * (D / 64) + w; tw[e] = word(x.v[k / 4], k % 4); }
    uint32_t lo01[4], hi01[4], lo23[4], hi23[4];
    widen((tw[0] & 0x0F0F0F0Fu) | ((tw[1] << 4) & 0xF0F0F0F0u), lo01);
    widen(((tw[0] >> 4) & 0x0F0F0F0Fu) | (tw[1] & 0xF0F0F0F0u), hi01);
    widen((tw[2] & 0x0F0F0F0Fu) | ((tw[3] << 4) & 0xF0F0F0F0u), lo23);
    widen(((tw[2] >> 4) & 0x0F0F0F0Fu) | (tw[3] & 0xF0F0F0F0u), hi23);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      T* to = vt + ((long long)h * 128 + g * (D / 8) + 8 * w + 2 * k) * t_cap + t0 + 4 * j;
      *reinterpret_cast<uint2*>(to) = make_uint2(to_t(times(lo01[k], s01)), to_t(times(lo23[k], s23)));
      *reinterpret_cast<uint2*>(to + t_cap) = make_uint2(to_t(times(hi01[k], s01)), to_t(times(hi23[k], s23)));
    }
  }
  if (D == 64)
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint2*>(vt + ((long long)h * 128 + 64 + g * 8 + i) * t_cap + t0 + 4 * j) = make_uint2(0, 0);
}

template <typename T, int D, int NB> int launch(const Fp4Args& a, int total_rows, int sms, cudaStream_t stream) {
  using S = Shape<D, NB>;
  static bool ready[64] = {}, weights_ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fp4_attention_kernel<T, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) { msgl_set_error("paged_attention_fp4 shared memory", e); return MSGL_CUDA_ERROR; }
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  msgl_launch(fp4_attention_kernel<T, D, NB>, dim3(a.workers / kWarps), dim3(kWarps * 32), S::smem, stream, a);
  MSGL_CHECK_LAUNCH("paged_attention_fp4");
  // a row's parts are some workers / (requests * key heads * row tiles): up to four for a warp
  const long long rows = (long long)total_rows * a.hq, each = (long long)a.workers * a.row_tile / (rows > 0 ? rows : 1);
  if (each < 8) msgl_launch(fp4_join_kernel<T, D, 1>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, a, total_rows);
  else if (each < 16) msgl_launch(fp4_join_kernel<T, D, 2>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a, total_rows);
  else msgl_launch(fp4_join_kernel<T, D, 8>, dim3((unsigned)rows), dim3(256), 0, stream, a, total_rows);
  MSGL_CHECK_LAUNCH("paged_attention_fp4 join");
  if (a.weights != nullptr) {
    using W = WeightsShape<D, (NB > 1)>;
    if (dev < 0 || dev >= 64 || !weights_ready[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(fp4_weights_kernel<T, D, (NB > 1)>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::smem);
      if (e != cudaSuccess) { msgl_set_error("paged_attention_fp4 weights shared memory", e); return MSGL_CUDA_ERROR; }
      if (dev >= 0 && dev < 64) weights_ready[dev] = true;
    }
    msgl_launch(fp4_weights_kernel<T, D, (NB > 1)>, dim3(sms * W::ctas), dim3(kWarps * 32), W::smem, stream, a);
    MSGL_CHECK_LAUNCH("paged_attention_fp4 weights");
  }
  return MSGL_OK;
}

int row_blocks(int d, int rows) { return rows <= 8 ? 1 : rows <= 16 || d == 256 ? 2 : 4; }

int device_sms() {
  static int sms[64] = {};
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && sms[dev]) return sms[dev];
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev >= 0 && dev < 64) sms[dev] = n;
  return n;
}

int* status_word() {
  static int* word[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && word[dev] != nullptr) return word[dev];
  int* p = nullptr;
  cudaGetSymbolAddress((void**)&p, g_fp4_status);
  if (dev >= 0 && dev < 64) word[dev] = p;
  return p;
}

int worker_count(int d, int nb) {
  return device_sms() * ctas_of(d, nb) * kWarps;
}

}  // namespace

// fp32 words of the workspace: the parts, the line (64 bits each), the rows' sums with weights.
MSGL_API long long msgl_attention_fp4_workspace(int total_rows, int B, int hq, int hk, int d, int max_q, int weighed) {
  if (hk <= 0) return 0;
  const int nb = row_blocks(d, max_q * (hq / hk));
  const long long parts = 2ll * worker_count(d, nb) * nb * 8 * (d + 4);
  return parts + 2ll * ((B < kMost ? B : kMost) + 2) + (weighed ? (long long)total_rows * hq : 0);
}

MSGL_API int msgl_attention_fp4(const void* q, void* out, const void* pool, const void* table, long long table_stride, int width,
                                const void* cu_q, const void* lens, const void* k_head, const void* v_head, void* weights,
                                void* workspace, int total_rows, int B, int hq, int hk, int d, int page_size, int pages, int max_q,
                                int window, float scale, int dtype, cudaStream_t stream) {
  if (B <= 0 || total_rows <= 0) return MSGL_OK;
  if (hk <= 0 || hq <= 0 || hq % hk || (d != 64 && d != 128 && d != 256) || page_size <= 0 || page_size % kTile ||
      (uintptr_t)pool % 16 || (uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)workspace % 16 || width <= 0 || max_q <= 0 ||
      (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("paged_attention_fp4: heads of 64, 128 or 256 channels, pages of whole tiles of 16 tokens, 16-bit queries");
    return MSGL_BAD_ARG;
  }
  const int nb = row_blocks(d, max_q * (hq / hk)), workers = worker_count(d, nb);
  int* status = status_word();
  float* ws = (float*)workspace;
  const long long parts = 2ll * workers * nb * 8 * (d + 4);
  for (int b0 = 0; b0 < B; b0 += kMost) {
    Fp4Args a{};
    a.B = B - b0 < kMost ? B - b0 : kMost;
    a.q = q; a.out = out; a.pool = (const uint8_t*)pool;
    a.table = (const int32_t*)table + b0 * table_stride; a.table_stride = table_stride; a.width = width;
    a.cu_q = (const int32_t*)cu_q + b0; a.lens = (const int32_t*)lens + b0;
    a.k_head = (const float*)k_head; a.v_head = (const float*)v_head; a.weights = (float*)weights;
    a.parts = ws; a.line = (long long*)(ws + parts);
    a.lse = weights != nullptr ? ws + parts + 2ll * ((B < kMost ? B : kMost) + 2) : nullptr;
    a.hq = hq; a.hk = hk; a.group = hq / hk; a.page_size = page_size; a.per = page_size / kTile; a.pages = pages; a.window = window;
    a.row_tile = 8 * nb; a.workers = workers; a.scale = scale; a.status = status;
    int rc = MSGL_BAD_ARG;
    const int sms = device_sms();
#define RUN(T, D, N) rc = launch<T, D, N>(a, total_rows, sms, stream)
#define WIDTHS(T)                                                                                                          \
  if (d == 64) { if (nb == 1) RUN(T, 64, 1); else if (nb == 2) RUN(T, 64, 2); else RUN(T, 64, 4); }                         \
  else if (d == 128) { if (nb == 1) RUN(T, 128, 1); else if (nb == 2) RUN(T, 128, 2); else RUN(T, 128, 4); }                \
  else { if (nb == 1) RUN(T, 256, 1); else RUN(T, 256, 2); }
    if (dtype == MSGL_BF16) { WIDTHS(__nv_bfloat16) } else { WIDTHS(__half) }
#undef WIDTHS
#undef RUN
    if (rc != MSGL_OK) return rc;
  }
  return MSGL_OK;
}

MSGL_API int msgl_gather_fp4(const void* pool, const void* table, long long table_stride, int width, void* kc, void* vt, const void* blk_req,
                             const void* req_info, long long t_cap, int t_pad, int hk, int d, int page_size, int pages, int dtype,
                             cudaStream_t stream) {
  if (t_pad <= 0) return MSGL_OK;
  if (hk <= 0 || (d != 64 && d != 128) || page_size <= 0 || page_size % kTile || (uintptr_t)pool % 16 || t_pad % 128 || t_pad > t_cap ||
      width <= 0 || (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("gather of a 4-bit pool: heads of 64 or 128 channels, blocks of 128 rows");
    return MSGL_BAD_ARG;
  }
  Fp4Args a{};
  a.pool = (const uint8_t*)pool; a.table = (const int32_t*)table; a.table_stride = table_stride; a.width = width;
  a.hk = hk; a.page_size = page_size; a.per = page_size / kTile; a.pages = pages;
  const int tiles = t_pad / kTile;
  const dim3 grid((tiles + 7) / 8, hk);
#define GATHER(T, D) msgl_launch(fp4_gather_kernel<T, D>, grid, dim3(256), 0, stream, a, (T*)kc, (T*)vt, (const int*)blk_req, (const int*)req_info, t_cap, tiles)
  if (dtype == MSGL_BF16) { if (d == 64) GATHER(__nv_bfloat16, 64); else GATHER(__nv_bfloat16, 128); }
  else { if (d == 64) GATHER(__half, 64); else GATHER(__half, 128); }
#undef GATHER
  MSGL_CHECK_LAUNCH("gather of a 4-bit pool");
  return MSGL_OK;
}

MSGL_API int msgl_attention_fp4_status(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_fp4_status, sizeof(int));
  if (reset && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_fp4_status, &z, sizeof(int));
  }
  return v;
}
