// Causal attention over the paged K/V pool of 4 bits (kv_fp4.cuh).
//
// A unit is a tile of rows of one request and key head, a row being a (query position, head of the group) pair, with all 16-token
// tiles that its request's rows see. The tiles of all units in a line are dealt evenly to the CTAs of the GPU, and a CTA's tiles
// two by two to its warps, each of which fetches its own into a ring (bulk copies of 18 D bytes) and keeps the softmax of the
// unit it is in. Where a unit ends the warps' sums are joined in shared memory. Units that a CTA has whole are written at
// once; of the others the parts go to the workspace, and the CTA that brings the last one joins them, in the order of the line.
//
// Both products take the cache as their first operand (rows: 16 tokens, or 16 channels), so a row tile is 8 queries wide and
// no product is spent on more rows than a group of 8 heads has: S^T = K Q^T, O^T = V^T P^T. Codes go e2m1 -> f16 (one
// conversion for two) and are multiplied by their scale, which is exact (2 + 4 significant bits). Queries are scaled to
// powers of two around 2^10 and taken as f16: exact for bf16 and fp16 values down to 2^-24 of a row's largest. Sums, running
// maximum and sum of the softmax are fp32. Probabilities go into the second product as f16 (11 bits) after a factor of 2^7,
// so that they are normal numbers down to 2^-21 of the largest; the maximum moves only when a score passes it by 2^8, which
// the factor leaves room for (2^15).
//
// Bound: a warp's own chain of instructions. A tile of 16 tokens of 128 channels takes a warp about 290, of which 209 widen and
// multiply: 64 conversions and 64 products with scales for 4096 values are what 4 bits cost over 8. The 12 warps that fit on an SM
// issue 0.56 of them a cycle and scheduler (issue slots 56 % busy, the ALU pipe 53 %, neither full), and an SM takes 15 bytes a clock of
// the 23 that DRAM has for it. B200, in a graph: 4 requests of 70 to 120 thousand tokens, 8 key heads of 128, 103 us, 4.3 TB/s; 256 of
// 500 to 2300 120 us, 3.4 TB/s; 64 of them 40 us, 2.7 TB/s (4 us until the first tiles come, 5 for the joins). Tried on the first: 16 warps an SM with 128 registers in place of 12 with 168 (105 to 107),
// 20 with 96 (spills, 127), the next pair's scores between this pair's values (105), parts joined by a second kernel (105), by all
// warps of the last CTA (101, but the 64 requests 43).
#include "kv_fp4.cuh"
#include "ptx.cuh"

using namespace msgl;
using namespace msgl::fp4;
using namespace msgl::ptx;

namespace {

constexpr int kWarps = 4;            // of a CTA
constexpr int kMost = 256;           // requests of a launch
constexpr int kFewTiles = 8;         // a CTA gets at least so many tiles: a pair for each warp
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
  float* parts;             // [2 * workers][blocks of 8 rows][D / 16 + 1 times 16 bytes of a lane][32 lanes]
  int* arrived;             // [workers]: parts of the unit that begins in a worker's share and goes on; zeros between calls
  int width, B, hq, hk, group, page_size, per, pages, window, row_tile, row_shift, workers;   // per: tiles of a page; row_tile: 2^row_shift
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
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
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
  __device__ __forceinline__ void rows_to(const Fp4Args& a, int row, int row_end) {
    q0 = row;
    q_len = row_end - row;
    row_tiles = (max(q_len, 0) * a.group + a.row_tile - 1) >> a.row_shift;
  }
};
// In shared memory: first tile of every request, the total behind them; first rows, lengths, tiles in sight.
struct Line {
  long long first[kMost + 1];
  int row[kMost + 1], n[kMost], tile0[kMost], tiles[kMost];
  int piece[kMost + 1];     // first piece of every request, where units are cut into pieces of `cut` tiles
  int cut;                  // else 0
  __device__ __forceinline__ Request request(const Fp4Args& a, int b) const {
    Request r;
    r.rows_to(a, row[b], row[b + 1]);
    r.n = n[b];
    r.tile0 = tile0[b];
    r.tiles = tiles[b];
    return r;
  }
};

// Sum of v over the CTA's threads in front of this one; `all`: over all of them.
template <typename V> __device__ __forceinline__ V scan(V v, V* sums, V& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  V before = incl - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    before += w < warp ? sums[w] : V(0);
    all += sums[w];
  }
  return before;
}

// `few` > 0: units may be cut into pieces of their own. The tiles of all units are dealt evenly then only if there are many: a
// CTA with the end of one unit and the beginning of another has two units to wait for, which counts where they are short.
// B200, us, dealt -> cut when the cut was added, 32 query and 8 key heads of 128: one request of 700 tokens 16.4 -> 12.4, 8 of 100 to 300
// 16.6 -> 12.5 (in a graph, both 10.2 now).
__device__ __forceinline__ void lay_line(const Fp4Args& a, Line& line, bool whole_rows, int few) {
  __shared__ long long sums[kWarps];
  __shared__ int sums32[2][kWarps];
  constexpr int PER = kMost / (kWarps * 32);
  long long cost[PER], mine = 0, total;
  int units[PER], tiles[PER], my_units = 0, all_units;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = (int)threadIdx.x * PER + i;
    cost[i] = 0;
    units[i] = tiles[i] = 0;
    if (b < a.B) {
      const int row = a.cu_q[b], row_end = a.cu_q[b + 1], len = a.lens[b];
      Request r;
      r.rows_to(a, row, row_end);
      r.n = min(max(len, 0), a.width * a.page_size);
      const int lo = a.window > 0 ? max(0, r.n - r.q_len - a.window + 1) : 0;
      r.tile0 = lo / kTile;
      r.tiles = r.q_len > 0 && r.n > lo ? (r.n + kTile - 1) / kTile - r.tile0 : 0;
      line.row[b] = row;
      line.n[b] = r.n;
      line.tile0[b] = r.tile0;
      line.tiles[b] = r.tiles;
      if (b == a.B - 1) line.row[a.B] = row_end;
      tiles[i] = r.tiles;
      units[i] = r.tiles > 0 ? a.hk * (whole_rows ? 1 : r.row_tiles) : 0;
      cost[i] = (long long)r.tiles * units[i];
    }
    mine += cost[i];
    my_units += units[i];
  }
  long long before = scan(mine, sums, total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = (int)threadIdx.x * PER + i;
    if (b < a.B) line.first[b] = before;
    before += cost[i];
    if (b == a.B - 1) line.first[a.B] = before;
  }
  int cut = 0;
  if (few > 0) {
    scan(my_units, sums32[0], all_units);
    if (all_units <= a.workers / 2 && total < 3ll * few * a.workers) {
      // so many pieces at most: one more for each unit than tiles / cut
      cut = max(few, (int)((total + a.workers - all_units - 1) / (a.workers - all_units)));
      int pieces = 0, all;
#pragma unroll
      for (int i = 0; i < PER; ++i) pieces += units[i] * ((tiles[i] + cut - 1) / cut);
      int at = scan(pieces, sums32[1], all);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int b = (int)threadIdx.x * PER + i;
        if (b < a.B) line.piece[b] = at;
        at += units[i] * ((tiles[i] + cut - 1) / cut);
        if (b == a.B - 1) line.piece[a.B] = at;
      }
    }
  }
  if (threadIdx.x == 0) line.cut = cut;
  __syncthreads();
}

// Divisions of 64 bits are calls; most lines are shorter than 2^32 tiles.
__device__ __forceinline__ long long quotient(long long x, int y) {
  return (x >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)y) : x / y;
}

// Worker w of W has tiles [begin(w), begin(w + 1)): `base`, and one more for the first `extra`.
struct Deal {
  long long base;
  int workers, extra;
  __device__ __forceinline__ Deal(long long total, int most, int few) {
    workers = (int)max(1ll, min((long long)most, quotient(total, few)));
    base = quotient(total, workers);
    extra = (int)(total - base * workers);
  }
  __device__ __forceinline__ long long begin(int w) const { return w * base + min(w, extra); }
  __device__ __forceinline__ int owner(long long at) const {
    const long long big = (base + 1) * extra;
    if ((base >> 31) == 0) return (int)(at < big ? quotient(at, (int)base + 1) : extra + quotient(at - big, max((int)base, 1)));
    return (int)(at < big ? at / (base + 1) : extra + (at - big) / base);
  }
};
// Worker w's piece of a unit: its tiles, and the workers that have the unit.
struct Piece {
  long long begin;
  int count, w0, w1;
  __device__ __forceinline__ Piece(const Line& line, int B, int w) {
    count = 0;
    if (w >= line.piece[B]) return;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (line.piece[mid] <= w) lo = mid; else hi = mid - 1;
    }
    const int tiles = line.tiles[lo], cut = line.cut, each = (tiles + cut - 1) / cut, at = w - line.piece[lo], unit = at / each;
    w0 = line.piece[lo] + unit * each;
    w1 = w0 + each - 1;
    begin = line.first[lo] + (long long)unit * tiles + (w - w0) * cut;
    count = min(cut, tiles - (w - w0) * cut);
  }
};

// A place in the line: a row tile (rt) of a key head of request b, and a tile of 16 tokens: sub of the page in column col of
// the block table. Steps take no divisions.
struct Walk {
  int b, head, rt, tile, col, sub;
  Request r;
  __device__ __forceinline__ void place(const Fp4Args& a) {
    col = r.tile0 + tile;
    sub = 0;
    if (a.per > 1) {
      const int t = col;
      col = t / a.per;
      sub = t - col * a.per;
    }
  }
  __device__ __forceinline__ void start_unit(const Fp4Args& a) {
    tile = 0;
    place(a);
  }
  __device__ __forceinline__ void seek(const Fp4Args& a, const Line& line, long long at, bool whole_rows) {
    int lo = 0, hi = a.B - 1;                   // the last request that starts at or before `at` has it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (line.first[mid] <= at) lo = mid; else hi = mid - 1;
    }
    b = lo;
    r = line.request(a, b);
    const long long o = at - line.first[b];
    head = (int)quotient(o, max(r.tiles, 1));
    tile = (int)(o - (long long)head * r.tiles);
    rt = 0;
    if (!whole_rows && r.row_tiles > 1) {
      const int unit = head;
      head = unit / r.row_tiles;
      rt = unit - head * r.row_tiles;
    }
    place(a);
  }
  // on to the next unit that has tiles
  __device__ __forceinline__ void next_unit(const Fp4Args& a, const Line& line, bool whole_rows) {
    if (!whole_rows && ++rt < r.row_tiles) { start_unit(a); return; }
    rt = 0;
    if (++head == a.hk) {
      head = 0;
      do ++b; while (b < a.B - 1 && line.first[b] == line.first[b + 1]);
      r = line.request(a, min(b, a.B - 1));
    }
    start_unit(a);
  }
  // true where another unit begins
  __device__ __forceinline__ bool next(const Fp4Args& a, const Line& line, bool whole_rows) {
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
// Lane 4 g + j has channels j D / 4 .. of row g.
template <typename T, int D>
__device__ __forceinline__ void fetch_query(const Fp4Args& a, const Request& r, int head, int row, int lane, Vec8<T> (&raw)[D / 32]) {
  const bool there = row < r.q_len * a.group;
  const int pos = there ? row / a.group : 0;
  const T* src = reinterpret_cast<const T*>(a.q) + ((long long)(r.q0 + pos) * a.hq + head * a.group + (there ? row - pos * a.group : 0)) * D
                 + (lane & 3) * (D / 4);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    *reinterpret_cast<uint4*>(&raw[i]) = make_uint4(0, 0, 0, 0);
    if (there) raw[i] = *reinterpret_cast<const Vec8<T>*>(src + 8 * i);
  }
}
// ... as the second operand of S^T, scaled by a power of two (a negative scale of the scores is the query's sign). Returns
// what the row's scores have to be multiplied by.
template <typename T, int D>
__device__ __forceinline__ float scale_query(const Fp4Args& a, const Vec8<T> (&raw)[D / 32], uint32_t (&qf)[D / 8]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int ex = (int)(__float_as_uint(top) >> 23);            // 0: zeros; 255: infinite
  const int up = top > 0.f && ex < 255 ? min(max(137 - ex, -126), 126) : 0;
  const float f = copysignf(__uint_as_float((uint32_t)(127 + up) << 23), a.scale);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float x[8];
    unpack8(raw[i], x);
#pragma unroll
    for (int e = 0; e < 4; ++e) qf[4 * i + e] = f16x2(x[2 * e] * f, x[2 * e + 1] * f);
  }
  return __uint_as_float((uint32_t)(127 - up) << 23);
}
template <typename T, int D>
__device__ __forceinline__ float load_query(const Fp4Args& a, const Request& r, int head, int row, int lane, uint32_t (&qf)[D / 8]) {
  Vec8<T> raw[D / 32];
  fetch_query<T, D>(a, r, head, row, lane, raw);
  return scale_query<T, D>(a, raw, qf);
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
        for (int nb = 0; nb < NB; ++nb) {
          if (w == 0 && c == 0) mma_first(s[nb], a0, a1, a2, a3, qf[nb][0], qf[nb][1]);
          else mma(s[nb], a0, a1, a2, a3, qf[nb][4 * w + 2 * c], qf[nb][4 * w + 2 * c + 1]);
        }
      }
    }
  }
}

// CTAs on an SM: what registers (without spilling the loop's values) and shared memory allow
__host__ __device__ constexpr int ctas_of(int d, int nb) { return d == 256 || nb > 1 ? 2 : d == 128 ? 3 : 4; }

template <int D, int NB> struct Shape {
  static constexpr int stages = D == 64 ? 4 : D == 128 ? 3 : 2;        // of two tiles
  static constexpr int ring = kWarps * stages * 2 * Tile<D>::bytes;
  static constexpr int record = (D / 16 + 1) * 512;                    // a warp's sums of 8 rows: 16 bytes of a lane at a time
  static constexpr int bars = ring + (kWarps - 1) * record, flag = bars + kWarps * stages * 8, line = flag + 16;
  static constexpr int smem = line + (int)sizeof(Line);
  static constexpr int ctas = ctas_of(D, NB);
  static_assert(ctas * (smem + 1024 + 64) <= 228 * 1024, "shared memory of an SM");
};

template <typename T, int D, int NB>
__global__ void __launch_bounds__(kWarps * 32, Shape<D, NB>::ctas) fp4_attention_kernel(const Fp4Args a) {
  using S = Shape<D, NB>;
  constexpr int STAGES = S::stages, BYTES = Tile<D>::bytes;
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint8_t* ring = smem + warp * STAGES * 2 * BYTES;
  float4* records = reinterpret_cast<float4*>(smem + S::ring);
  const uint32_t bar = smem_u32(smem + S::bars) + warp * STAGES * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::flag);
  Line& line = *reinterpret_cast<Line*>(smem + S::line);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bar + 8 * s, 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_wait();
  // With weights to come the next kernel starts when this one has ended, and so does the one behind it: kernels that wait for
  // this one in places that its CTAs leave, here and there, come out of step with it (48 requests: 110 us, so 87).
  if (a.weights == nullptr) pdl_trigger();
  lay_line(a, line, false, kFewTiles);
  // rows of requests without a token in sight belong to no unit
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const Request r = line.request(a, b);
    if (r.tiles > 0) continue;
    for (long long i = threadIdx.x; i < (long long)max(r.q_len, 0) * a.hq * (D / 8); i += kWarps * 32)
      reinterpret_cast<uint4*>(a.out)[(long long)r.q0 * a.hq * (D / 8) + i] = make_uint4(0, 0, 0, 0);
  }
  const int worker = blockIdx.x;
  const Deal deal(line.first[a.B], a.workers, kFewTiles);
  long long at = 0;
  int total = 0, piece0 = 0, piece1 = 0;      // tiles; workers of the unit where units are cut
  if (line.cut > 0) {
    const Piece p(line, a.B, worker);
    at = p.begin;
    total = p.count;
    piece0 = p.w0;
    piece1 = p.w1;
  } else if (worker < deal.workers) {
    at = deal.begin(worker);
    total = (int)(deal.begin(worker + 1) - at);
  }
  if (total <= 0) return;

  // Tiles come in pairs, dealt to the warps in turn, a stage for each. Lane i finds the places of the warp's pairs i, 32 + i,
  // ... and fetches them: no step along the line for each tile.
  const int pairs = ((total + 1) / 2 - warp + kWarps - 1) / kWarps;
  const uint8_t *mine0 = nullptr, *mine1 = nullptr;
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched % 32 == 0) {
      const int p = 2 * (warp + kWarps * (fetched + lane));
      Walk w;
      w.seek(a, line, at + min(p, total - 1), false);
      const int page0 = w.page(a);                   // (both pages are asked for before one is used)
      mine0 = w.address<D>(a, 0);
      if (p + 1 < total) w.next(a, line, false);
      const int page1 = w.page(a);
      mine1 = w.address<D>(a, page1);
      mine0 += (long long)page0 * a.hk * a.per * BYTES;
    }
    if (lane == fetched % 32) {
      const bool both = 2 * (warp + kWarps * fetched) + 1 < total;
      const uint32_t full = bar + 8 * stage, to = smem_u32(ring + stage * 2 * BYTES);
      mbar_expect_tx(full, both ? 2 * BYTES : BYTES);
      bulk_load(to, mine0, BYTES, full);
      if (both) bulk_load(to + BYTES, mine1, BYTES, full);
    }
    ++fetched;
  };
  const int g = lane >> 2, j = lane & 3;
  Walk get;
  get.seek(a, line, at, false);
  Vec8<T> raw[NB][D / 32];       // the queries of the first unit are asked for ahead of its tiles
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) fetch_query<T, D>(a, get.r, get.head, get.rt * a.row_tile + nb * 8 + g, lane, raw[nb]);
  for (int s = 0; s < STAGES && s < pairs; ++s) fetch(s);

  int done = 0, pair = 2 * warp, stage = 0;       // done: tiles of the CTA's units so far; pair: first tile of the warp's next pair
  uint32_t phase = 0;
  bool ok = true;
  while (done < total) {
    // ---- one unit, or this CTA's part of it
    const int first = get.tile, head = get.head, row0 = get.rt * a.row_tile;
    const int count = min(total - done, get.r.tiles - first);       // tiles of it that this CTA has
    const Request r = get.r;
    const int rows = min(a.row_tile, r.q_len * a.group - row0);
    uint32_t qf[NB][D / 8];
    float2 c[NB];                // factors of the scores of rows 2 j and 2 j + 1, above 0
    const float kh = fabsf(a.scale) * kLog2e * (a.k_head != nullptr ? a.k_head[head] : 1.f);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float back = scale_query<T, D>(a, raw[nb], qf[nb]);
      c[nb].x = fmaxf(kh * __shfl_sync(0xffffffffu, back, 8 * j), 1e-37f);
      c[nb].y = fmaxf(kh * __shfl_sync(0xffffffffu, back, 8 * j + 4), 1e-37f);
    }
    // m: running maxima; base: minus what is taken from a score in the exponent; limit: the score, without its factor, from
    // which the maximum moves
    float o[NB][D / 16][4], m[NB][2], limit[NB][2];
    float2 base[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
      m[nb][0] = m[nb][1] = limit[nb][0] = limit[nb][1] = -INFINITY;
      base[nb] = make_float2(kUp, kUp);
      l[nb] = make_float2(0.f, 0.f);
    }
    // tokens [lo_all, hi_all) are seen by all rows
    const int pos0 = r.n - r.q_len + row0 / a.group, pos1 = r.n - r.q_len + (row0 + rows - 1) / a.group;
    const int hi_all = pos0 + 1, lo_all = a.window > 0 ? pos1 - a.window + 1 : 0;

    const int end = done + count;
    auto arrive = [&](int st, uint32_t ph) { return __all_sync(0xffffffffu, mbar_wait(bar + 8 * st, ph, abort_flag, a.status, 401)); };
    while (pair < end && ok) {
      ok = arrive(stage, phase);
      if (!ok) break;
      const uint8_t* tile = ring + stage * 2 * BYTES;
      // of the pair's tiles one may be another unit's: `from` .. `to` are the tokens of this one, tok0 is the pair's first
      const int from = max(done - pair, 0) * kTile, to = min(2, end - pair) * kTile;
      const int tok0 = (r.tile0 + first + pair - done) * kTile;
      if (tok0 + from <= pos1) {                                     // else rows behind these see it
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
            move |= fmaxf(fmaxf(s[0][nb][k], s[0][nb][2 + k]), fmaxf(s[1][nb][k], s[1][nb][2 + k])) > limit[nb][k];
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float factor = k ? c[nb].y : c[nb].x;
              float top = fmaxf(fmaxf(s[0][nb][k], s[0][nb][2 + k]), fmaxf(s[1][nb][k], s[1][nb][2 + k])) * factor;
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              top = fmaxf(top, m[nb][k]);
              const float f = m[nb][k] == top ? 1.f : exp2_fast(m[nb][k] - top);
              m[nb][k] = top;
              limit[nb][k] = (top + kSlack) / factor;
              (k ? base[nb].y : base[nb].x) = kUp - (top == -INFINITY ? 0.f : top);
              (k ? l[nb].y : l[nb].x) *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[nb][i][k] *= f; o[nb][i][2 + k] *= f; }
            }
          }
        }
        uint32_t p[2][NB][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float2 e = fma2(make_float2(s[u][nb][2 * h], s[u][nb][2 * h + 1]), c[nb], base[nb]);
              e.x = exp2_fast(e.x);
              e.y = exp2_fast(e.y);
              l[nb] = add2(l[nb], e);
              p[u][nb][h] = transpose8(f16x2(e.x, e.y));
            }
        Raw<D> x[2];
        load_values<D>(tile, lane, x[0]);
        load_values<D>(tile + BYTES, lane, x[1]);
        // values of tokens that no row sees may be anything; a NaN that only some rows see must not reach the others
        uint32_t nan_mask = 0;       // bit 8 u + 4 i + e: token 4 j + e of tile u has no number in block i of the lane's channels
        if (ragged) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < (D == 256 ? 2 : 1); ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((x[u].vs[i] >> (8 * e) & 0x7F) == 0x7F) {
                  nan_mask |= 1u << (8 * u + 4 * i + e);
                  x[u].vs[i] &= ~(0xFFu << (8 * e));
                }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {                  // words of 8 channels of the lane: 4 products
            const int i = D == 256 ? w / 2 : 0;
            const uint32_t s01 = widen_e4m3(x[u].vs[i]), s23 = widen_e4m3(x[u].vs[i] >> 16);
            uint32_t tw[4];                                    // of tokens 4 j .. 4 j + 3
#pragma unroll
            for (int e = 0; e < 4; ++e) { const int k = e * (D / 64) + w; tw[e] = word(x[u].v[k / 4], k % 4); }
            uint32_t lo01[4], hi01[4], lo23[4], hi23[4];       // pairs of tokens of the even and of the odd channels
            widen((tw[0] & 0x0F0F0F0Fu) | ((tw[1] << 4) & 0xF0F0F0F0u), lo01);
            widen(((tw[0] >> 4) & 0x0F0F0F0Fu) | (tw[1] & 0xF0F0F0F0u), hi01);
            widen((tw[2] & 0x0F0F0F0Fu) | ((tw[3] << 4) & 0xF0F0F0F0u), lo23);
            widen(((tw[2] >> 4) & 0x0F0F0F0Fu) | (tw[3] & 0xF0F0F0F0u), hi23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a0 = times(lo01[k], s01), a1 = times(hi01[k], s01), a2 = times(lo23[k], s23), a3 = times(hi23[k], s23);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) mma(o[nb][4 * w + k], a0, a1, a2, a3, p[u][nb][0], p[u][nb][1]);
            }
          }
        }
        if (ragged && __any_sync(0xffffffffu, nan_mask != 0)) {
          for (int jj = 0; jj < 4; ++jj) {
            const uint32_t bits = __shfl_sync(0xffffffffu, nan_mask, 4 * g + jj);
            for (int t = 0; t < 8; ++t) {                      // tile t / 4, token t % 4 of the lane
              const int tok = t / 4 * kTile + 4 * jj + t % 4;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int pos = r.n - r.q_len + (row0 + nb * 8 + 2 * j + k) / a.group;
                  const bool seen = tok < min(min(pos + 1, r.n) - tok0, to) && tok >= from &&
                                    !(a.window > 0 && tok0 + tok <= pos - a.window);
#pragma unroll
                  for (int i = 0; i < D / 16; ++i)
                    if (seen && (bits >> (t / 4 * 8 + (D == 256 ? i / 8 * 4 : 0) + t % 4) & 1)) o[nb][i][k] = o[nb][i][2 + k] = NAN;
                }
            }
          }
        }
      }
      if (to < 2 * kTile && end < total) break;          // the next unit has the pair's other tile
      __syncwarp();
      if (fetched < pairs) fetch(stage);
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      pair += 2 * kWarps;
    }
    done = end;
    if (done < total) {                                              // the next unit's queries are asked for
      get.next_unit(a, line, false);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) fetch_query<T, D>(a, get.r, get.head, get.rt * a.row_tile + nb * 8 + g, lane, raw[nb]);
    }

    // ---- the warps' sums are joined in the first one, 8 rows at a time
    auto write = [&](float4* to, int nb) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) to[i * 32 + lane] = make_float4(o[nb][i][0], o[nb][i][1], o[nb][i][2], o[nb][i][3]);
      to[D / 16 * 32 + lane] = make_float4(m[nb][0], m[nb][1], l[nb].x, l[nb].y);
    };
    auto join = [&](const float4 (&x)[D / 16 + 1], int nb) {
      const float4 ml = x[D / 16];
      float f[2], h[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float other = k ? ml.y : ml.x, top = fmaxf(m[nb][k], other);
        f[k] = m[nb][k] == top ? 1.f : exp2_fast(m[nb][k] - top);
        h[k] = other == top ? 1.f : exp2_fast(other - top);
        m[nb][k] = top;
      }
      l[nb] = make_float2(l[nb].x * f[0] + ml.z * h[0], l[nb].y * f[1] + ml.w * h[1]);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[nb][i][0] = o[nb][i][0] * f[0] + x[i].x * h[0];
        o[nb][i][1] = o[nb][i][1] * f[1] + x[i].y * h[1];
        o[nb][i][2] = o[nb][i][2] * f[0] + x[i].z * h[0];
        o[nb][i][3] = o[nb][i][3] * f[1] + x[i].w * h[1];
      }
    };
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      for (int d = 4; d < 32; d <<= 1) {
        l[nb].x += __shfl_xor_sync(0xffffffffu, l[nb].x, d);
        l[nb].y += __shfl_xor_sync(0xffffffffu, l[nb].y, d);
      }
      if (nb * 8 >= rows) break;
      __syncthreads();                                   // the records have been read
      if (warp > 0) write(records + (warp - 1) * (S::record / 16), nb);
      __syncthreads();
      if (warp == 0) {
#pragma unroll 1
        for (int w = 0; w < kWarps - 1; ++w) {
          float4 x[D / 16 + 1];
#pragma unroll
          for (int i = 0; i <= D / 16; ++i) x[i] = records[w * (S::record / 16) + i * 32 + lane];
          join(x, nb);
        }
      }
    }
    if (warp == 0) {         // (after a wait that ran out too: the counters have to come out even)
      bool finish = first == 0 && count == r.tiles;
      if (!finish) {
        // the unit's other parts: of the workers from the one that it begins with to the one that it ends with
        const long long u0 = at + (end - count) - first;
        const int w0 = line.cut > 0 ? piece0 : deal.owner(u0), w1 = line.cut > 0 ? piece1 : deal.owner(u0 + r.tiles - 1);
        float4* part = reinterpret_cast<float4*>(a.parts);
        auto place = [&](int w, int nb) { return part + ((long long)(2 * w + (w == w0 ? 1 : 0)) * NB + nb) * (S::record / 16); };
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          if (nb * 8 < rows) write(place(worker, nb), nb);
        __syncwarp();
        int before = 0;
        if (lane == 0) {
          __threadfence();
          before = atomicAdd(a.arrived + w0, 1);
        }
        before = __shfl_sync(0xffffffffu, before, 0);
        finish = before == w1 - w0;
        if (finish) {
          __threadfence();
          if (lane == 0) a.arrived[w0] = 0;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            if (nb * 8 >= rows) break;
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb] = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nb][i][0] = o[nb][i][1] = o[nb][i][2] = o[nb][i][3] = 0.f;
            float4 x[2][D / 16 + 1];                     // one part is on its way while the other is added
            auto ask = [&](int w, float4 (&x)[D / 16 + 1]) {
              const float4* from = place(min(w, w1), nb) + lane;
#pragma unroll
              for (int i = 0; i <= D / 16; ++i) x[i] = __ldcg(from + i * 32);
            };
            ask(w0, x[0]);
#pragma unroll 1
            for (int w = w0; w <= w1; w += 2) {
              ask(w + 1, x[1]);
              join(x[0], nb);
              if (w == w1) break;
              ask(w + 2, x[0]);
              join(x[1], nb);
            }
          }
        }
      }
      if (finish) {
        // rows 2 j and 2 j + 1 of every block: channels g D / 8 .. (D / 8 of them)
        const float vh = a.v_head != nullptr ? a.v_head[head] : 1.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = nb * 8 + 2 * j + k;
            if (row >= rows) continue;
            const float sum = k ? l[nb].y : l[nb].x, f = sum > 0.f || sum != sum ? vh / sum : 0.f;
            const int qi = (row0 + row) / a.group;
            const long long to = (long long)(r.q0 + qi) * a.hq + head * a.group + (row0 + row - qi * a.group);
            T* dst = reinterpret_cast<T*>(a.out) + to * D + g * (D / 8);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) { y[2 * e] = o[nb][4 * i + e][k] * f; y[2 * e + 1] = o[nb][4 * i + e][2 + k] * f; }
              store8(dst + 8 * i, y);
            }
            if (a.lse != nullptr && g == 0) a.lse[to] = (m[nb][k] == -INFINITY ? 0.f : m[nb][k]) - kUp + log2f(sum);
          }
        }
      }
    }
  }
  if (!ok) {     // copies may be in flight: they land before the shared memory goes
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

// What the rows give every token: the keys once more, with the rows' final maxima and sums. A tile's keys go through all rows of
// their (request, key head) pair, so a token's sum is taken by one lane in one order. MANY false: up to 8 rows, in registers;
// warps deal out the tiles of all pairs (should a request have more rows than the caller said, its row tiles follow each other and
// add to a token in any order). MANY: CTAs do; the pair's queries lie in shared memory, `chunk` blocks of 8 rows at
// a time, and the warps take the CTA's tiles in turn. A warp has four tiles' keys under way. Bound: instructions; 48 requests of 900
// to 5000 tokens 33 us beside the attention's 52 (one chain of products 35; five CTAs an SM the same). The scores that the first kernel has could be kept instead, 32 bytes written and
// read for a token and 4 query heads against the 72 of its key, but in a captured step they would need memory for the longest request
// that may come.
template <int D, bool MANY> struct WeightsShape {
  static constexpr int stages = 4, key_bytes = 9 * D;                  // codes and scales
  static constexpr int chunk = !MANY ? 0 : D == 256 ? 4 : 16;          // blocks of 8 rows
  static constexpr int ctas = D == 256 ? 2 : MANY ? 3 : 4;
  static constexpr int ring = kWarps * stages * key_bytes, bars = ring, slots = bars + kWarps * stages * 8;
  static constexpr int flag = slots + kWarps * stages * 4, line = flag + 16, queries = (line + (int)sizeof(Line) + 15) / 16 * 16;
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
  Line& line = *reinterpret_cast<Line*>(smem + S::line);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(bar + 8 * s, 1);
    if (warp == 0) *abort_flag = 0;
    fence_barrier_init();
  }
  pdl_wait();
  lay_line(a, line, MANY, 0);
  const Deal deal(line.first[a.B], MANY ? gridDim.x : gridDim.x * kWarps, MANY ? 8 : 4);
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
      w.seek(a, line, first + (long long)min(fetched + lane, count - 1) * step, MANY);
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
  // weights that the two rows 2 j, 2 j + 1 of a block give tokens of rows g and g + 8. A row that is not there has an infinite
  // log of its sum.
  auto given = [&](const Request& r, int row0, int tok0, const float (&s)[4], float2 c, float2 e, float& s0, float& s1) {
    const float2 minus = make_float2(-e.x, -e.y);
    float2 p0 = fma2(make_float2(s[0], s[1]), c, minus), p1 = fma2(make_float2(s[2], s[3]), c, minus);
    const int ahead = r.n - r.q_len;                       // position of the first row
    if (tok0 + kTile - 1 > ahead || (a.window > 0 && tok0 <= r.n - 1 - a.window)) {     // else all rows see all tokens
      const int posA = ahead + (row0 + 2 * j) / a.group, posB = ahead + (row0 + 2 * j + 1) / a.group;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = tok0 + token_of(g, i >> 1), pos = i & 1 ? posB : posA;
        const bool seen = tok <= min(pos, r.n - 1) && !(a.window > 0 && tok <= pos - a.window);
        if (!seen) (i < 2 ? (i & 1 ? p0.y : p0.x) : (i & 1 ? p1.y : p1.x)) = -INFINITY;
      }
    }
    s0 += exp2_fast(p0.x) + exp2_fast(p0.y);
    s1 += exp2_fast(p1.x) + exp2_fast(p1.y);
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
  get.seek(a, line, at, MANY);
  if constexpr (!MANY) {
    count = (int)(end - at);
    for (int s = 0; s < min(STAGES, count); ++s) fetch();
    __syncwarp();
    uint32_t qf[D / 8];
    float2 c = {}, e = {};
    bool fresh = true;
    while (done < count) {
      if (fresh) {
        const float back = load_query<T, D>(a, get.r, get.head, 8 * get.rt + g, lane, qf);
        const float kh = fabsf(a.scale) * kLog2e * (a.k_head != nullptr ? a.k_head[get.head] : 1.f);
        c = make_float2(kh * __shfl_sync(0xffffffffu, back, 8 * j), kh * __shfl_sync(0xffffffffu, back, 8 * j + 4));
        e = make_float2(lse_of(get.r, get.head, 8 * get.rt + 2 * j), lse_of(get.r, get.head, 8 * get.rt + 2 * j + 1));
      }
      next_keys();
      if (!ok) break;
      float s[4], s2[4];               // two chains of products
      mma_first(s, k[0][0], k[0][1], k[0][2], k[0][3], qf[0], qf[1]);
      mma_first(s2, k[1][0], k[1][1], k[1][2], k[1][3], qf[2], qf[3]);
#pragma unroll
      for (int i = 2; i < D / 16; i += 2) {
        mma(s, k[i][0], k[i][1], k[i][2], k[i][3], qf[2 * i], qf[2 * i + 1]);
        mma(s2, k[i + 1][0], k[i + 1][1], k[i + 1][2], k[i + 1][3], qf[2 * i + 2], qf[2 * i + 3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += s2[i];
      const int tok0 = (get.r.tile0 + get.tile) * kTile;
      float s0 = 0.f, s1 = 0.f;
      given(get.r, 8 * get.rt, tok0, s, c, e, s0, s1);
      give(get.r, tok0, s0, s1);
      if (done < count) fresh = get.next(a, line, false);
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
        const int blocks = min(S::chunk, (rows - row0 + 15) / 16 * 2);   // an even number: rows that are not there weigh nothing
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
          for (int nb = 0; nb < blocks; nb += 2) {         // two chains of products side by side
            float s[2][4];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint4 q = queries[((nb + u) * (D / 32) + i) * 32 + lane];
                if (i == 0) mma_first(s[u], k[0][0], k[0][1], k[0][2], k[0][3], q.x, q.y);
                else mma(s[u], k[2 * i][0], k[2 * i][1], k[2 * i][2], k[2 * i][3], q.x, q.y);
                mma(s[u], k[2 * i + 1][0], k[2 * i + 1][1], k[2 * i + 1][2], k[2 * i + 1][3], q.z, q.w);
              }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float4 c = *reinterpret_cast<const float4*>(rowc + (nb + u) * 8 + 2 * j);
              given(r, row0 + (nb + u) * 8, tok0, s[u], make_float2(c.x, c.z), make_float2(c.y, c.w), s0, s1);
            }
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
  for (int e = 0; e < 4; ++e)                  // what lies behind the request may be anything; fp4_prompt_nans_kernel puts NaNs back
    if (tok0 + 4 * j + e >= n || (x.vs[0] >> (8 * e) & 0x7F) == 0x7F) x.vs[0] &= ~(0xFFu << (8 * e));
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

// NaN values of a prompt step. The product of probabilities and values would give one that only later rows of a block see to the
// earlier ones too (0 * NaN), so the gather leaves zeros in their place and this kernel writes the NaNs over the output of the rows
// that see them: 16 channels of a value each. Without any, which is nearly always, it reads a tile's value scales and is done: 553 us of two prompts
// of some 2000 rows behind prefixes stay 553.
template <typename T, int D> __global__ void __launch_bounds__(256)
fp4_prompt_nans_kernel(const Fp4Args a, T* __restrict__ out, const int* __restrict__ items, int n_items, const int* __restrict__ blk_req,
                       const int* __restrict__ req_info, int tiles) {
  pdl_enter();
  const int lane = threadIdx.x & 31, id = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (id >= tiles) return;
  const int h = blockIdx.y, t0 = id * kTile, req = blk_req[t0 >> 7];
  const int tok0 = t0 - req_info[3 * req] + req_info[3 * req + 2], n = req_info[3 * req + 1];
  if (tok0 >= n) return;
  const int page = min(max(a.table[(long long)req * a.table_stride + min(tok0 / a.page_size, a.width - 1)], 0), a.pages - 1);
  const uint8_t* tile = a.pool + ((long long)(page * a.hk + h) * a.per + tok0 / kTile % a.per) * Tile<D>::bytes;
  uint32_t bad = 0;                            // lanes 4 b .. 4 b + 3: tokens whose block b is NaN
  if (lane < D / 4) {
    const uint32_t sf = *reinterpret_cast<const uint32_t*>(tile + Tile<D>::v_sf + 4 * lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 4 * (lane & 3) + e;
      if ((sf >> (8 * e) & 0x7F) == 0x7F && tok0 + t < n) bad |= 1u << t;
    }
  }
  if (!__any_sync(0xffffffffu, bad != 0)) return;
  bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
  bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
  for (int i = 0; i < n_items; ++i) {          // blocks of rows: first row, rows, first position, ., ., request
    const int* it = items + 8 * i;
    if (it[5] != req) continue;
    for (int row = 0; row < it[1]; ++row) {
      const int hi = it[2] + row - tok0, lo = a.window > 0 ? hi - a.window : -1;        // tokens lo + 1 .. hi of the tile are seen
      uint32_t seen = hi < 0 ? 0u : (2u << min(hi, 15)) - 1u;
      if (lo >= 0) seen &= ~((2u << min(lo, 15)) - 1u);
      if (lane < D / 4 && (bad & seen))
        for (int g = 0; g < a.group; ++g)      // four channels a lane
          *reinterpret_cast<uint2*>(out + ((long long)(it[0] + row) * a.hq + h * a.group + g) * D + 4 * lane) = make_uint2(0x7FFF7FFFu, 0x7FFF7FFFu);
    }
  }
}

template <typename T, int D, int NB> int launch(const Fp4Args& a, cudaStream_t stream) {
  using S = Shape<D, NB>;
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fp4_attention_kernel<T, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) { msgl_set_error("paged_attention_fp4 shared memory", e); return MSGL_CUDA_ERROR; }
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  msgl_launch(fp4_attention_kernel<T, D, NB>, dim3(a.workers), dim3(kWarps * 32), S::smem, stream, a);
  MSGL_CHECK_LAUNCH("paged_attention_fp4");
  return MSGL_OK;
}

// Blocks of 8 rows in a row tile: two, so that keys and values are widened once for 16 rows, where the registers have room.
// B200, us: some 25 rows each of 3 requests of 5 to 9 thousand tokens, 32 heads of 128, with weights: four blocks (spilling) 154,
// two 126; four warps of 16 rows each that share widened tiles through shared memory the same as two (they wait for one another);
// 16 heads a key head of 256, 20 requests of 2 to 6 thousand: two (spilling) 83, one 58.
int row_blocks(int d, int rows) { return rows <= 8 || d == 256 ? 1 : 2; }

template <typename T, int D, bool MANY> int launch_weights(const Fp4Args& a, int sms, cudaStream_t stream) {
  using W = WeightsShape<D, MANY>;
  static bool ready[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(fp4_weights_kernel<T, D, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::smem);
    if (e != cudaSuccess) { msgl_set_error("paged_attention_fp4 weights shared memory", e); return MSGL_CUDA_ERROR; }
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  msgl_launch(fp4_weights_kernel<T, D, MANY>, dim3(sms * W::ctas), dim3(kWarps * 32), W::smem, stream, a);
  MSGL_CHECK_LAUNCH("paged_attention_fp4 weights");
  return MSGL_OK;
}

long long parts_words(int d, int nb, int workers) { return 2ll * workers * nb * (d / 16 + 1) * 128; }

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
  return device_sms() * ctas_of(d, nb);
}

}  // namespace

// fp32 words of the workspace: the parts; the rows' sums with weights. `workers`: words of `arrived`.
MSGL_API long long msgl_attention_fp4_workspace(int total_rows, int hq, int hk, int d, int max_q, int weighed, int* workers) {
  if (hk <= 0) return 0;
  const int nb = row_blocks(d, max_q * (hq / hk)), most = worker_count(d, nb);
  *workers = most;
  return parts_words(d, nb, most) + (weighed ? (long long)total_rows * hq : 0);
}

MSGL_API int msgl_attention_fp4(const void* q, void* out, const void* pool, const void* table, long long table_stride, int width,
                                const void* cu_q, const void* lens, const void* k_head, const void* v_head, void* weights,
                                void* workspace, void* arrived, int total_rows, int B, int hq, int hk, int d, int page_size, int pages, int max_q,
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
  for (int b0 = 0; b0 < B; b0 += kMost) {
    Fp4Args a{};
    a.B = B - b0 < kMost ? B - b0 : kMost;
    a.q = q; a.out = out; a.pool = (const uint8_t*)pool;
    a.table = (const int32_t*)table + b0 * table_stride; a.table_stride = table_stride; a.width = width;
    a.cu_q = (const int32_t*)cu_q + b0; a.lens = (const int32_t*)lens + b0;
    a.k_head = (const float*)k_head; a.v_head = (const float*)v_head; a.weights = (float*)weights;
    a.parts = ws; a.arrived = (int*)arrived;
    a.lse = weights != nullptr ? ws + parts_words(d, nb, workers) : nullptr;
    a.hq = hq; a.hk = hk; a.group = hq / hk; a.page_size = page_size; a.per = page_size / kTile; a.pages = pages; a.window = window;
    a.row_tile = 8 * nb; a.row_shift = nb == 1 ? 3 : 4; a.workers = workers; a.scale = scale; a.status = status;
    int rc = MSGL_BAD_ARG;
    const int sms = device_sms();
    const bool many = max_q * (hq / hk) > 8;
#define RUN(T, D)                                                                                                            \
  do {                                                                                                                       \
    rc = nb == 1 ? launch<T, D, 1>(a, stream) : launch<T, D, D == 256 ? 1 : 2>(a, stream);                                    \
    if (rc == MSGL_OK && weights != nullptr)                                                                                 \
      rc = many ? launch_weights<T, D, true>(a, sms, stream) : launch_weights<T, D, false>(a, sms, stream);                  \
  } while (0)
    if (dtype == MSGL_BF16) { if (d == 64) RUN(__nv_bfloat16, 64); else if (d == 128) RUN(__nv_bfloat16, 128); else RUN(__nv_bfloat16, 256); }
    else { if (d == 64) RUN(__half, 64); else if (d == 128) RUN(__half, 128); else RUN(__half, 256); }
#undef RUN
    if (rc != MSGL_OK) return rc;
  }
  return MSGL_OK;
}

MSGL_API int msgl_attn_prefill_tc(const void* q, long long q_row_stride, void* out, const void* k_pool, const void* v_pool, void* kc,
                                  void* vt, long long t_cap, int t_pad, const void* items, int n_items, const void* blk_req,
                                  const void* req_info, const void* block_table, int bt_stride, const void* k_scale, const void* v_scale,
                                  int total_q, int hq, int hk, int d, int page_size, int kv_fp8, float scale, int window, int chunk,
                                  float softcap, const void* gate, long long ldg, const void* bias, int entries, int zero,
                                  const void* sink, int all_values, int pos_form, int dtype, cudaStream_t stream);

// A prompt step: the rows in sight to 16 bits (`kc`, `vt`: 128 hk t_cap elements each), the tensor-core kernel, NaN values. `items`,
// `blk_req`, `req_info`: the tables of the step, as there.
MSGL_API int msgl_prompt_fp4(const void* q, void* out, const void* pool, const void* table, long long table_stride, int width, void* kc,
                             void* vt, long long t_cap, int t_pad, const void* items, int n_items, const void* blk_req,
                             const void* req_info, const void* k_head, const void* v_head, int total_q, int hq, int hk, int d,
                             int page_size, int pages, int window, int pos_form, float scale, int dtype, cudaStream_t stream) {
  if (t_pad <= 0 || n_items <= 0 || total_q <= 0) return MSGL_OK;
  if (hk <= 0 || hq <= 0 || hq % hk || (d != 64 && d != 128) || page_size <= 0 || page_size % kTile || (uintptr_t)pool % 16 ||
      (uintptr_t)out % 16 || t_pad % 128 || t_pad > t_cap || width <= 0 || (dtype != MSGL_BF16 && dtype != MSGL_F16)) {
    msgl_set_error_text("prompts over a 4-bit pool: heads of 64 or 128 channels, blocks of 128 rows");
    return MSGL_BAD_ARG;
  }
  Fp4Args a{};
  a.pool = (const uint8_t*)pool; a.table = (const int32_t*)table; a.table_stride = table_stride; a.width = width;
  a.hq = hq; a.hk = hk; a.group = hq / hk; a.page_size = page_size; a.per = page_size / kTile; a.pages = pages; a.window = window;
  const int tiles = t_pad / kTile;
  const dim3 grid((tiles + 7) / 8, hk);
#define GATHER(T, D) msgl_launch(fp4_gather_kernel<T, D>, grid, dim3(256), 0, stream, a, (T*)kc, (T*)vt, (const int*)blk_req, (const int*)req_info, t_cap, tiles)
  if (dtype == MSGL_BF16) { if (d == 64) GATHER(__nv_bfloat16, 64); else GATHER(__nv_bfloat16, 128); }
  else { if (d == 64) GATHER(__half, 64); else GATHER(__half, 128); }
#undef GATHER
  MSGL_CHECK_LAUNCH("gather of a 4-bit pool");
  const int rc = msgl_attn_prefill_tc(q, (long long)hq * d, out, nullptr, nullptr, kc, vt, t_cap, t_pad, items, n_items, blk_req, req_info,
                                      table, 0, k_head, v_head, total_q, hq, hk, d, page_size, 2, scale, window, 0, 0.f, nullptr, 0,
                                      nullptr, 0, 0, nullptr, 0, pos_form, dtype, stream);
  if (rc != MSGL_OK) return rc;
#define NANS(T, D) msgl_launch(fp4_prompt_nans_kernel<T, D>, grid, dim3(256), 0, stream, a, (T*)out, (const int*)items, n_items, (const int*)blk_req, (const int*)req_info, tiles)
  if (dtype == MSGL_BF16) { if (d == 64) NANS(__nv_bfloat16, 64); else NANS(__nv_bfloat16, 128); }
  else { if (d == 64) NANS(__half, 64); else NANS(__half, 128); }
#undef NANS
  MSGL_CHECK_LAUNCH("NaN values of a prompt");
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
