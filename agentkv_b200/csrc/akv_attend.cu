// akv_attend.cu — attention of one new token of each sequence over the paged
// pool, split over the sequences' lengths and joined.
//
// For a row's query head with scores x_j = scale * q . k_j over the positions
// j that take part, the output is sum_j e^(x_j) v_j / sum_j e^(x_j).  A piece
// of the positions gives m = max_j x_j, l = sum_j e^(x_j - m) and
// o = sum_j e^(x_j - m) v_j; pieces join by m = max m_i,
// l = sum_i e^(m_i - m) l_i, o = sum_i e^(m_i - m) o_i.  Exponentials are
// taken to base 2 with log2(e) in the scale.
//
// What bounds it: each key and value is read once for the whole group of
// query heads that shares it (4 * group flops per 2-byte element pair), so the
// time is the pool's bytes over the HBM rate.
//
// Work: a pair is one row with one key head (or a part of its query heads,
// where they are more than a product has columns), and its work is the row's
// chunks of 64 positions.  All pairs' chunks, one behind another, are dealt to
// the CTAs in equal contiguous ranges, whatever the rows' lengths are (the host
// does not know them, and a captured launch replays with others).  A pair
// inside one range is finished there; of one that crosses ranges each CTA
// leaves a piece in scratch, and the last CTA to do so joins them (by 20s
// where there are more).
#include <climits>

#include "akv_paged.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 16;               // positions per warp and step
constexpr int kChunk = kTile * kWarps;  // positions per CTA and step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Where nothing has been seen yet (a finite number: differences stay numbers).
constexpr float kLowest = -3.402823466e38f;
// A running maximum is raised only once a score lies this far above it (the
// sums are the same for any m, so long as 2^(x - m) stays in range: at most
// 2^8 here), which spares most steps the reduction over the lanes.
constexpr float kLazy = 8.0f;
// Weights as fp16 numbers: those have no step below 2^-24, so weights that are
// to be in range must not lie near 1.  m is held kHalfBelow below the maximum and
// raised once a score lies kHalfLazy above m: weights reach 2^15 at most (65,504 is
// the largest number), the maximum's own is 2^11 at least, and what has no step
// is under 2^-36 of it.
constexpr float kHalfBelow = 11.0f;
constexpr float kHalfLazy = 15.0f;
constexpr int kLeast = 2;                  // chunks per CTA: a piece costs as much as one or two
constexpr int kFan = 20;                   // pieces that are joined at a time
constexpr int kMaxCtas = kFan * kFan * 2;  // two levels of joining

struct AttendParams {
  AkvLayer kv;
  AkvTables tab;
  const int32_t* selected;
  int32_t keep;
  const void* q;
  int64_t q_row, q_head;
  void* out;
  int64_t out_row, out_head;
  float* lse;
  int32_t group, parts;  // query heads per key head, and the pairs that they make
  float scale_log2;
  int32_t window;
  float* pieces;
  int32_t* arrived;  // [3 * gridDim.x], zero between launches
  AkvStatus* st;
};

// Row s: positions [lo, n) take part, in chunks [first, first + chunks) of the
// row (of its selected blocks, where there is a selection).
struct Extent {
  int32_t n, lo, first, chunks;
};

AKV_DEV Extent row_extent(const AttendParams& p, int32_t s) {
  Extent e;
  e.n = akv_held(p.tab, p.kv.bs_log2, s);
  e.lo = p.window > 0 && e.n > p.window ? e.n - p.window : 0;
  if (p.selected) {
    const int32_t blocks = (e.n + (1 << p.kv.bs_log2) - 1) >> p.kv.bs_log2;
    const int32_t taken = (blocks < p.keep ? blocks : p.keep) << p.kv.bs_log2;
    e.first = 0;
    e.chunks = (taken + kChunk - 1) / kChunk;
  } else {
    e.first = e.lo / kChunk;
    e.chunks = (e.n + kChunk - 1) / kChunk - e.first;
  }
  return e;
}

// A run of positions that lie behind one another in one block: 8, or 1 where
// blocks are smaller.
struct Run {
  int32_t id;   // the block, kNone: none
  int32_t pos;  // the first position
  static constexpr int32_t kNone = INT_MIN;
};

// The run at token `tok` of the row's list (of its selected blocks, where there is a
// selection).
AKV_DEV Run find_run(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t tok) {
  const int bl = p.kv.bs_log2;
  const int32_t blocks = (e.n + (1 << bl) - 1) >> bl;
  Run run = {Run::kNone, 0};
  int32_t place = tok >> bl;
  if (place >= blocks) return run;
  if (p.selected) {
    if (place >= p.keep) return run;
    place = p.selected[(static_cast<int64_t>(s) * p.kv.heads + h) * p.keep + place];
    if (place < -1 || place >= blocks) akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, place, blocks);
    if (place < 0 || place >= blocks) return run;
  }
  if (((place + 1ll) << bl) <= e.lo) return run;
  run.pos = (place << bl) + (tok & ((1 << bl) - 1));
  run.id = p.tab.ids[s * p.tab.stride + place];
  return run;
}

// The block of a run, if the pool has it.
AKV_DEV bool run_ok(const AttendParams& p, const Run& run, int32_t s) {
  if (static_cast<uint32_t>(run.id) < static_cast<uint32_t>(p.kv.total)) return true;
  if (run.id != Run::kNone) akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, run.id, p.kv.total);
  return false;
}

// Which of the `count` positions from `pos` take part.
AKV_DEV uint32_t taking_part(const Extent& e, int32_t pos, int count) {
  const int low = max(0, min(count, e.lo - pos)), high = max(low, min(count, e.n - pos));
  return ((1u << high) - 1) & ~((1u << low) - 1);
}

// A warp's view of the runs under its tiles: lane i holds where one lies, for
// the next 16 (or 2) tiles.
struct Cursor {
  int64_t off;    // bytes from the layer's K of this head
  uint32_t part;  // which of the run's positions take part
  uint32_t full;  // bit i: all of lane i's run does
  int32_t from;   // the first chunk that the runs are for

  AKV_DEV static int run_log2(int bs_log2) { return bs_log2 >= 3 ? 3 : 0; }
  AKV_DEV static int runs(int bs_log2) { return kTile >> run_log2(bs_log2); }  // per tile

  AKV_DEV void refill(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t chunk, int32_t end,
                      int warp, int lane) {
    from = chunk;
    const int bl = p.kv.bs_log2, rl = run_log2(bl), per = runs(bl);
    const int32_t c = chunk + lane / per;
    Run run = {Run::kNone, 0};
    if (c < end) run = find_run(p, e, s, h, c * kChunk + warp * kTile + (lane % per << rl));
    const bool ok = run_ok(p, run, s);
    off = ok ? run.id * p.kv.page_bytes + static_cast<int64_t>(run.pos & ((1 << bl) - 1)) * p.kv.row_bytes : 0;
    part = ok ? taking_part(e, run.pos, 1 << rl) : 0;
    full = __ballot_sync(kFullWarp, part == (1u << (1 << rl)) - 1);
  }
  // The lane that holds the run of position r (0..15) of chunk's tile.
  AKV_DEV int lane_of(int bs_log2, int32_t chunk, int r) const {
    return (chunk - from) * runs(bs_log2) + (r >> run_log2(bs_log2));
  }
  AKV_DEV bool covers(int bs_log2, int32_t chunk) const { return (chunk - from + 1) * runs(bs_log2) <= 32; }
  // Where position r of chunk's tile lies (all lanes call).
  AKV_DEV int64_t row(const AttendParams& p, int32_t chunk, int r) const {
    const int bl = p.kv.bs_log2, in = r & ((1 << run_log2(bl)) - 1);
    return __shfl_sync(kFullWarp, off, lane_of(bl, chunk, r)) + in * p.kv.row_bytes;
  }
  // Which of the tile's 16 positions take part (bit r).
  AKV_DEV uint32_t valid(const AttendParams& p, int32_t chunk, int lane) const {
    const int bl = p.kv.bs_log2, r = lane & 15, per = runs(bl);
    const uint32_t mine = full >> (chunk - from) * per;
    if (per == 2 && (mine & 3) == 3) return 0xffff;
    const uint32_t bits = __shfl_sync(kFullWarp, part, lane_of(bl, chunk, r));
    return __ballot_sync(kFullWarp, bits >> (r & ((1 << run_log2(bl)) - 1)) & 1) & 0xffff;
  }
};

// ── tensor-core engine: 16-bit types, head dims that are whole 16-byte words ─
// A warp takes 16 positions at a time with m16n8k16 products: S^T = K Q^T
// (positions x heads), then O^T += V^T P^T (dimensions x heads); 8 query
// heads are one product's width, so no row of a product is padding for a group
// of 8.  tcgen05 has 64 rows at least and wants its operands in shared memory:
// with 4 to 16 query heads it would copy every byte once more to run
// mostly empty.  Here the fragments come from global memory straight into
// registers: the order of the head dimensions in Q K^T and of the rows of V^T
// is free, so each lane loads 16 consecutive bytes of a row and the products
// take them in that order (lane 4 g + c holds dimensions 32 i + 8 c .. + 7 of
// key rows g and g + 8; of V, dimensions 64 i + 8 g .. + 7 of positions 2 c,
// 2 c + 1, 2 c + 8, 2 c + 9).  The next tile's keys are loaded as soon as this
// one's have been used, this one's values while the scores are computed.
// (Measured on 256 rows of 4,096 positions, 4.3 GB, where a plain read of the
// same blocks takes 615 us: 16-byte asynchronous copies into shared memory
// 846 us, bulk copies of whole blocks 765 us: their issue and the reads
// from shared memory held the warps up more than the memory did; this form
// 639-667 us, 6.4-6.7 TB/s.  One row of 200,001 positions 138-144 us, 5.7-5.9 TB/s.)
template <typename T>
struct Pack2;
template <>
struct Pack2<__half> {
  AKV_DEV static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  AKV_DEV static float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  AKV_DEV static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Pack2<__nv_bfloat16> {
  AKV_DEV static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  AKV_DEV static float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
  AKV_DEV static void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

AKV_DEV uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 2^x, off by 2^-22 of it at most, and 0 below 2^-126.  Both are far under half a step
// of the 16-bit outputs (2^-8 of a value in bf16, 2^-11 in fp16); the 32-bit engine takes exp2f.
AKV_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

AKV_DEV uint4 ld16(const char* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
AKV_DEV uint2 ld8(const char* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }

// Compiled for kD = 64, 96, 128 and 256; the dimensions between (kExact false) take the
// next one's products with zeros behind their own words.  At 168 registers the form of
// 128 spills 28 bytes a thread (68 for the dimensions between), that of 256 at 255
// registers 16 (160); the others none.
template <typename T, int kD, int kN, bool kExact>
struct MmaEngine {
  using Type = T;
  static constexpr int kDim = kExact ? kD : 0;
  static constexpr int kCols = 8 * kN;     // query heads per pair
  static constexpr int kCtas = kD <= 128 && kN == 1 ? 3 : (kD <= 128 ? 2 : 1);
  static constexpr int kKi = kD / 32;      // 16-byte words of a key row per lane
  static constexpr int kVi = kD / 64;      // the same of a value row,
  static constexpr bool kVr = kD % 64 != 0;  // and 8 bytes more
  static constexpr int kMt = kD / 16;      // output tiles of 16 dimensions
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr float kBelow = kHalf ? kHalfBelow : 0.f;  // m lies this far below the maximum at most
  static constexpr float kRaise = kHalf ? kHalfLazy : kLazy;

  uint4 q[kN][kKi];
  uint4 ka[kKi], kb[kKi];
  uint4 v[4][kVi];
  uint2 vr[4];
  float o[kN][kMt][4];
  float m[kN][2], l[kN][2];

  AKV_DEV static int row_of(const AttendParams& p) { return kExact ? kD * 2 : p.kv.row_bytes; }
  // Whether word w (of `bytes` bytes) of a row is one of its own.
  AKV_DEV static bool has(const AttendParams& p, int w, int bytes = 16) {
    return kExact || w * bytes < p.kv.row_bytes;
  }

  // Positions that take no part (bits of vm) are 0, whatever the block holds.
  AKV_DEV void load_k(const AttendParams& p, const Cursor& cur, const char* base, int32_t chunk, uint32_t vm,
                      int lane) {
    const int g = lane >> 2, c = lane & 3;
    const char *pa, *pb;
    if (p.kv.bs_log2 >= 3) {
      pa = base + __shfl_sync(kFullWarp, cur.off, (chunk - cur.from) * 2) + g * row_of(p);
      pb = base + __shfl_sync(kFullWarp, cur.off, (chunk - cur.from) * 2 + 1) + g * row_of(p);
    } else {
      pa = base + cur.row(p, chunk, g);
      pb = base + cur.row(p, chunk, g + 8);
    }
    pa += c * 16;
    pb += c * 16;
    if (kExact && vm == 0xffffu) {
#pragma unroll
      for (int i = 0; i < kKi; ++i) {
        ka[i] = ld16(pa + i * 64);
        kb[i] = ld16(pb + i * 64);
      }
    } else {
      const bool va = (vm >> g) & 1, vb = (vm >> (g + 8)) & 1;
#pragma unroll
      for (int i = 0; i < kKi; ++i) {
        ka[i] = va && has(p, i * 4 + c) ? ld16(pa + i * 64) : make_uint4(0, 0, 0, 0);
        kb[i] = vb && has(p, i * 4 + c) ? ld16(pb + i * 64) : make_uint4(0, 0, 0, 0);
      }
    }
  }

  AKV_DEV void load_v(const AttendParams& p, const Cursor& cur, const char* base, int32_t chunk, uint32_t vm,
                      int lane) {
    const int g = lane >> 2, c = lane & 3;
    const char* row[4];
    if (p.kv.bs_log2 >= 3) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        row[2 * half] = base + __shfl_sync(kFullWarp, cur.off, (chunk - cur.from) * 2 + half) + c * 2 * row_of(p);
        row[2 * half + 1] = row[2 * half] + row_of(p);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) row[x] = base + cur.row(p, chunk, 2 * c + (x & 1) + (x >> 1) * 8);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int r = 2 * c + (x & 1) + (x >> 1) * 8;
      if (vm == 0xffffu || ((vm >> r) & 1)) {
#pragma unroll
        for (int i = 0; i < kVi; ++i)
          v[x][i] = has(p, i * 8 + g) ? ld16(row[x] + i * 128 + g * 16) : make_uint4(0, 0, 0, 0);
        if (kVr) vr[x] = has(p, kVi * 16 + g, 8) ? ld8(row[x] + kVi * 128 + g * 8) : make_uint2(0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < kVi; ++i) v[x][i] = make_uint4(0, 0, 0, 0);
        if (kVr) vr[x] = make_uint2(0, 0);
      }
    }
  }

  AKV_DEV void values(int tile, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, const uint32_t (&hi)[kN][2],
                      const uint32_t (&lo)[kN][2]) {
    const uint32_t a0 = __byte_perm(x0, x1, 0x5410), a1 = __byte_perm(x0, x1, 0x7632);
    const uint32_t a2 = __byte_perm(x2, x3, 0x5410), a3 = __byte_perm(x2, x3, 0x7632);
#pragma unroll
    for (int n = 0; n < kN; ++n) Pack2<T>::mma(o[n][tile], a0, a1, a2, a3, hi[n][0], hi[n][1]);
#pragma unroll
    for (int n = 0; n < kN; ++n) Pack2<T>::mma(o[n][tile], a0, a1, a2, a3, lo[n][0], lo[n][1]);
  }

  // Chunks [a, b) of pair (s, h, part): this warp's tiles.
  AKV_DEV void run(const AttendParams& p, const Extent& ext, int32_t s, int32_t h, int32_t part, int32_t a, int32_t b,
                   int warp, int lane) {
    const int g = lane >> 2, c = lane & 3;
    const char* kbase = p.kv.base + h * p.kv.tile_bytes;
    const char* vbase = kbase + p.kv.kv_bytes;
    Cursor cur;
    cur.refill(p, ext, s, h, a, b, warp, lane);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int32_t head = part * kCols + n * 8 + g;
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + head) * p.q_head;
#pragma unroll
      for (int i = 0; i < kKi; ++i)
        q[n][i] = head < p.group && has(p, i * 4 + c) ? ld16(reinterpret_cast<const char*>(row + i * 32 + c * 8))
                                                      : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int t = 0; t < kMt; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][t][x] = 0.f;
      m[n][0] = m[n][1] = kLowest;
      l[n][0] = l[n][1] = 0.f;
    }
    uint32_t vm = cur.valid(p, a, lane);
    load_k(p, cur, kbase, a, vm, lane);
    for (int32_t chunk = a; chunk < b; ++chunk) {
      load_v(p, cur, vbase, chunk, vm, lane);
      float sc[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float odd[4] = {0.f, 0.f, 0.f, 0.f};  // two chains of products
        sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < kKi; ++i) {
          Pack2<T>::mma(sc[n], ka[i].x, kb[i].x, ka[i].y, kb[i].y, q[n][i].x, q[n][i].y);
          Pack2<T>::mma(odd, ka[i].z, kb[i].z, ka[i].w, kb[i].w, q[n][i].z, q[n][i].w);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[n][x] += odd[x];
      }
      const uint32_t now = vm;
      if (chunk + 1 < b) {
        if (!cur.covers(p.kv.bs_log2, chunk + 1)) cur.refill(p, ext, s, h, chunk + 1, b, warp, lane);
        vm = cur.valid(p, chunk + 1, lane);
        load_k(p, cur, kbase, chunk + 1, vm, lane);
      }
      float e[kN][4], above = 0.f;
      auto exponents = [&]() {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            e[n][x] = fmaf(sc[n][x], p.scale_log2, -m[n][x & 1]);
            if (now != 0xffff && !(now >> (g + (x >> 1) * 8) & 1)) e[n][x] = -INFINITY;
            above = fmaxf(above, e[n][x]);
          }
      };
      exponents();
      if (__any_sync(kFullWarp, above > kRaise)) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = m[n][x] + kBelow;
            if (now >> g & 1) top = fmaxf(top, sc[n][x] * p.scale_log2);
            if (now >> (g + 8) & 1) top = fmaxf(top, sc[n][x + 2] * p.scale_log2);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, off));
            top -= kBelow;
            const float by = exp2_fast(m[n][x] - top);
            m[n][x] = top;
            l[n][x] *= by;
#pragma unroll
            for (int t = 0; t < kMt; ++t) {
              o[n][t][x] *= by;
              o[n][t][x + 2] *= by;
            }
          }
        exponents();
      }
      // The weights go into the product as the sum of two 16-bit numbers:
      // one alone would be off by half a step of the type, as much as the
      // output's own rounding; the time is the memory's either way.  The two
      // are off by 2^-18 of the weight in bf16; in fp16 by 2^-24 of it and, where the
      // second is below the type's normal range, by 2^-25 (2^-36 of the largest weight).
      uint32_t hi[kN][2], lo[kN][2];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float w0 = exp2_fast(e[n][2 * x]), w1 = exp2_fast(e[n][2 * x + 1]);
          l[n][0] += w0;
          l[n][1] += w1;
          const uint32_t top = Pack2<T>::pack(w0, w1);
          const float2 r = Pack2<T>::unpack(top);
          hi[n][x] = transpose8x8(top);
          lo[n][x] = transpose8x8(Pack2<T>::pack(w0 - r.x, w1 - r.y));
        }
      }
#pragma unroll
      for (int i = 0; i < kVi; ++i) {
        values(4 * i + 0, v[0][i].x, v[1][i].x, v[2][i].x, v[3][i].x, hi, lo);
        values(4 * i + 1, v[0][i].y, v[1][i].y, v[2][i].y, v[3][i].y, hi, lo);
        values(4 * i + 2, v[0][i].z, v[1][i].z, v[2][i].z, v[3][i].z, hi, lo);
        values(4 * i + 3, v[0][i].w, v[1][i].w, v[2][i].w, v[3][i].w, hi, lo);
      }
      if (kVr) {
        values(4 * kVi + 0, vr[0].x, vr[1].x, vr[2].x, vr[3].x, hi, lo);
        values(4 * kVi + 1, vr[0].y, vr[1].y, vr[2].y, vr[3].y, hi, lo);
      }
    }
  }

  // This warp's sums: acc [kCols][dim], and m and l of each head.
  AKV_DEV void store(float* acc, float2* ml, int dim, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float sum = l[n][x];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(kFullWarp, sum, off);
        const int head = n * 8 + 2 * c + x;
        if (g == 0) ml[head] = make_float2(m[n][x], sum);
#pragma unroll
        for (int t = 0; t < kMt; ++t) {
          const int d = t < 4 * kVi ? (t >> 2) * 64 + g * 8 + 2 * (t & 3) : kVi * 64 + g * 4 + 2 * (t - 4 * kVi);
          if (kExact || d < dim)
            *reinterpret_cast<float2*>(acc + head * dim + d) = make_float2(o[n][t][x], o[n][t][x + 2]);
        }
      }
  }
};

// ── 32-bit engine: any type and head dim (up to 256) ───────────────────────
// Multiplies and adds in 32 bits, one row per pair.  kL lanes hold a row
// between them, kE consecutive dimensions of every kL kE each, so a warp has
// 32 / kL positions at a time; kU such steps give kU * kH partial scores per
// lane, which halving exchanges turn into one whole score (or a copy) per
// lane.  The next positions are loaded while these are computed.  What bounds it:
// latency, with 16 warps an SM (48 rows, window of 1,024, head dim 64: 35 us, 88 MB,
// 2.5 TB/s; 41 us with three CTAs an SM instead of four; 16 rows of 8,000 at 128
// dimensions 317 to 420 us, 3.3 to 2.5 TB/s).
template <typename T, int kE, int kJ, int kL, int kH>
struct SimtEngine {
  using Type = T;
  static constexpr int kDim = 0;
  static constexpr int kCols = kH;
  static constexpr int kX = kE * kJ;                      // dimensions per lane
  static constexpr int kCtas = kH * kX * kL >= 32 * 32 ? 2 : kH * kX <= 8 ? 4 : 3;
  static constexpr int kSub = 32 / kL;                    // positions at a time
  static constexpr int kU = kL / kH < 4 || kX > 4 ? 2 : 4;
  static constexpr int kVals = kU * kH;                   // scores at a time,
  static constexpr int kStep = kL / kVals;                // each held by this many lanes
  static constexpr int kPass = kU * kSub;                 // positions of a pass
  static_assert(kTile % kPass == 0 && kStep >= 1, "a tile is whole passes");
  using Word = AkvPack<T, kE>;

  float q[kH][kX], o[kH][kX];
  float m, l;  // of this lane's head, l over this lane's positions

  AKV_DEV static void load_row(Word (&x)[kJ], const char* row, int dim, bool ok, int at) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int d = (j * kL + at) * kE;
      x[j] = ok && d < dim ? akv_load<T, kE>(row + d * sizeof(T)) : Word{};
    }
  }

  AKV_DEV void load_pass(const AttendParams& p, const Cursor& cur, const char* kbase, int32_t chunk, uint32_t vm,
                         int r0, int lane, Word (&k)[kU][kJ], Word (&v)[kU][kJ]) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int r = r0 + u * kSub + lane / kL;
      const char* row = kbase + cur.row(p, chunk, r);
      load_row(k[u], row, p.kv.dim, (vm >> r) & 1, lane % kL);
      load_row(v[u], row + p.kv.kv_bytes, p.kv.dim, (vm >> r) & 1, lane % kL);
    }
  }

  AKV_DEV void compute(const AttendParams& p, uint32_t vm, int r0, int lane, const Word (&k)[kU][kJ],
                       const Word (&v)[kU][kJ]) {
    const int at = lane % kL, mine = at / kStep % kU;  // this lane's position of the kU
    float val[kVals];
#pragma unroll
    for (int n = 0; n < kH; ++n)
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          float x[kE];
          akv_unpack<T, kE>(x, k[u][j]);
#pragma unroll
          for (int i = 0; i < kE; ++i) d = fmaf(q[n][j * kE + i], x[i], d);
        }
        val[n * kU + u] = d;
      }
    // value i ends, whole, in lanes i * kStep ..: each exchange keeps the
    // half of the values that belongs to this lane's half
    int off = kL / 2;
#pragma unroll
    for (int w = kVals / 2; w >= 1; w >>= 1, off >>= 1) {
      const bool up = lane & off;
#pragma unroll
      for (int i = 0; i < w; ++i) {
        const float send = up ? val[i] : val[i + w];
        const float keep = up ? val[i + w] : val[i];
        val[i] = keep + __shfl_xor_sync(kFullWarp, send, off);
      }
    }
#pragma unroll
    for (int x = kStep / 2; x >= 1; x >>= 1) val[0] += __shfl_xor_sync(kFullWarp, val[0], x);
    const bool in = (vm >> (r0 + mine * kSub + lane / kL)) & 1;
    const float sc = val[0] * p.scale_log2;
    if (__any_sync(kFullWarp, in && sc > m + kLazy)) {
      float top = in ? fmaxf(sc, m) : m;
#pragma unroll
      for (int x = kStep; x < kStep * kU; x <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, x));
#pragma unroll
      for (int x = kL; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, x));
      const float by = exp2f(m - top);
      m = top;
      l *= by;
#pragma unroll
      for (int n = 0; n < kH; ++n) {
        const float f = __shfl_sync(kFullWarp, by, n * kU * kStep);
#pragma unroll
        for (int x = 0; x < kX; ++x) o[n][x] *= f;
      }
    }
    const float w = in ? exp2f(sc - m) : 0.f;
    l += w;
#pragma unroll
    for (int n = 0; n < kH; ++n)
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float f = __shfl_sync(kFullWarp, w, (lane & ~(kL - 1)) + (n * kU + u) * kStep);
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          float x[kE];
          akv_unpack<T, kE>(x, v[u][j]);
#pragma unroll
          for (int i = 0; i < kE; ++i) o[n][j * kE + i] = fmaf(f, x[i], o[n][j * kE + i]);
        }
      }
  }

  // Chunks [a, b) of pair (s, h, part): this warp's tiles.
  AKV_DEV void run(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t part, int32_t a, int32_t b,
                   int warp, int lane) {
#pragma unroll
    for (int n = 0; n < kH; ++n) {
      const int32_t head = part * kH + n;
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + head) * p.q_head;
      Word w[kJ];
      load_row(w, reinterpret_cast<const char*>(row), p.kv.dim, head < p.group, lane % kL);
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        float x[kE];
        akv_unpack<T, kE>(x, w[j]);
#pragma unroll
        for (int i = 0; i < kE; ++i) q[n][j * kE + i] = x[i];
      }
#pragma unroll
      for (int x = 0; x < kX; ++x) o[n][x] = 0.f;
    }
    m = kLowest;
    l = 0.f;
    const char* kbase = p.kv.base + h * p.kv.tile_bytes;
    Cursor cur;
    cur.refill(p, e, s, h, a, b, warp, lane);
    uint32_t vm = cur.valid(p, a, lane);
    Word k[kU][kJ], v[kU][kJ];
    load_pass(p, cur, kbase, a, vm, 0, lane, k, v);
    for (int32_t chunk = a; chunk < b; ++chunk) {
#pragma unroll 1
      for (int r0 = 0; r0 < kTile; r0 += kPass) {
        Word kn[kU][kJ], vn[kU][kJ];
        const uint32_t now = vm;
        const bool last = r0 + kPass >= kTile, more = !last || chunk + 1 < b;
        if (last && more) {
          if (!cur.covers(p.kv.bs_log2, chunk + 1)) cur.refill(p, e, s, h, chunk + 1, b, warp, lane);
          vm = cur.valid(p, chunk + 1, lane);
        }
        if (more) load_pass(p, cur, kbase, last ? chunk + 1 : chunk, vm, last ? 0 : r0 + kPass, lane, kn, vn);
        if (now >> r0 & ((1u << kPass) - 1)) compute(p, now, r0, lane, k, v);
        if (more) {
#pragma unroll
          for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              k[u][j] = kn[u][j];
              v[u][j] = vn[u][j];
            }
        }
      }
    }
  }

  AKV_DEV void store(float* acc, float2* ml, int dim, int lane) {
    float sum = l;
#pragma unroll
    for (int x = kStep; x < kStep * kU; x <<= 1) sum += __shfl_xor_sync(kFullWarp, sum, x);
#pragma unroll
    for (int x = kL; x < 32; x <<= 1) sum += __shfl_xor_sync(kFullWarp, sum, x);
    if (lane < kL && lane % (kU * kStep) == 0) ml[lane / (kU * kStep)] = make_float2(m, sum);
#pragma unroll
    for (int n = 0; n < kH; ++n)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          float x = o[n][j * kE + i];
#pragma unroll
          for (int w = kL; w < 32; w <<= 1) x += __shfl_xor_sync(kFullWarp, x, w);
          const int d = (j * kL + lane % kL) * kE + i;
          if (d < dim && lane < kL) acc[n * dim + d] = x;
        }
  }
};

// The factor that brings sums taken with maximum ml.x to maximum `to`; nothing
// (ml.y == 0) stays nothing.
AKV_DEV float join_factor(float2 ml, float to) { return ml.y == 0.f ? 0.f : exp2f(ml.x - to); }

template <typename T>
AKV_DEV void finish(const AttendParams& p, int32_t s, int32_t head, int d, float o, float l) {
  T* out = static_cast<T*>(p.out) + s * p.out_row + head * p.out_head;
  out[d] = from_f32<T>(l == 0.f ? 0.f : o / l);
}

AKV_DEV void finish_lse(const AttendParams& p, int32_t s, int32_t head, float m, float l) {
  if (p.lse)
    p.lse[static_cast<int64_t>(s) * p.kv.heads * p.group + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// A piece: [cols][dim] sums, then [cols] (m, l).
AKV_HD int64_t piece_floats(int cols, int dim) { return (static_cast<int64_t>(cols) * (dim + 2) + 3) / 4 * 4; }

// What a launch's CTAs agree on: unit u of `total` belongs to CTA cta_of(u).
struct Deal {
  int64_t total, ctas;
  AKV_DEV int64_t begin(int64_t c) const { return total * c / ctas; }
  AKV_DEV int64_t cta_of(int64_t u) const {
    int64_t c = u * ctas / total;
    while (begin(c + 1) <= u) ++c;
    while (begin(c) > u) --c;
    return c;
  }
};

template <class Eng>
__global__ void __launch_bounds__(kThreads, Eng::kCtas) k_attend(AttendParams p) {
  using T = typename Eng::Type;
  constexpr int kC = Eng::kCols;
  using Search = AkvRowSearch<kThreads>;
  extern __shared__ __align__(16) float acc[];  // [kWarps][kC][dim]
  __shared__ float2 ml[kWarps][kC];
  __shared__ float factor[kWarps][kC];
  __shared__ float2 joined[kC];
  __shared__ int32_t order;  // of this CTA's arrival
  __shared__ typename Search::Shared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dim = Eng::kDim ? Eng::kDim : p.kv.dim;
  const int64_t pairs = static_cast<int64_t>(p.kv.heads) * p.parts;  // of a row
  auto units = [&](int32_t s) -> int64_t { return row_extent(p, s).chunks * pairs; };

  int32_t s = 0;
  int64_t rest = 0, x = 0, end = 0;
  Deal deal;
  {
    Search search;
    search.scan(sh, p.tab.rows, units);
    deal.total = search.total;
    deal.ctas = min(static_cast<int64_t>(gridDim.x), (deal.total + kLeast - 1) / kLeast);
    if (blockIdx.x < deal.ctas) {
      x = deal.begin(blockIdx.x);
      end = deal.begin(blockIdx.x + 1);
      search.find(sh, x, units, s, rest);
    }
  }
  // rows that hold nothing, and lengths that no table can hold
  for (int32_t r = blockIdx.x; r < p.tab.rows; r += gridDim.x) {
    const int32_t n = akv_held(p.tab, p.kv.bs_log2, r);
    if (threadIdx.x == 0 && p.tab.lengths[r] != n)
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, r, p.tab.lengths[r], p.tab.width);
    if (n == 0) {
      const int32_t heads = p.kv.heads * p.group;
      for (int64_t i = threadIdx.x; i < static_cast<int64_t>(heads) * dim; i += kThreads)
        finish<T>(p, r, static_cast<int32_t>(i / dim), static_cast<int>(i % dim), 0.f, 0.f);
      for (int32_t i = threadIdx.x; i < heads; i += kThreads) finish_lse(p, r, i, 0.f, 0.f);
    }
  }
  while (x < end) {
    const Extent e = row_extent(p, s);
    if (rest >= e.chunks * pairs) {  // to the next row that holds something
      ++s;
      rest = 0;
      continue;
    }
    const int32_t pair = static_cast<int32_t>(rest / e.chunks);
    const int32_t a = static_cast<int32_t>(rest - static_cast<int64_t>(pair) * e.chunks);
    const int32_t n = static_cast<int32_t>(end - x < e.chunks - a ? end - x : e.chunks - a);
    const int32_t h = pair / p.parts, part = pair % p.parts;
    const bool whole = a == 0 && n == e.chunks;
    const int cols = min(kC, p.group - part * kC);
    const int32_t head0 = h * p.group + part * kC;
    {
      Eng eng;
      eng.run(p, e, s, h, part, e.first + a, e.first + a + n, warp, lane);
      eng.store(acc + warp * kC * dim, ml[warp], dim, lane);
    }
    __syncthreads();
    if (threadIdx.x < kC) {
      const int c = threadIdx.x;
      float top = kLowest, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w][c].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        factor[w][c] = join_factor(ml[w][c], top);
        sum += factor[w][c] * ml[w][c].y;
      }
      joined[c] = make_float2(top, sum);
    }
    __syncthreads();
    // the CTAs of the pair; a CTA's first piece may go on from the CTA before
    // it, its second begins in it
    const int64_t c0 = whole ? blockIdx.x : deal.cta_of(x - a);
    const int64_t c1 = whole ? blockIdx.x : deal.cta_of(x - a + e.chunks - 1);
    const int64_t size = piece_floats(kC, dim);
    auto slot = [&](int64_t c) { return p.pieces + (2 * c + (c == c0 ? 1 : 0)) * size; };
    float* const mine = slot(blockIdx.x);
    for (int i = threadIdx.x; i < cols * dim; i += kThreads) {
      const int c = i / dim;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (factor[w][c] != 0.f) sum = fmaf(factor[w][c], acc[w * kC * dim + i], sum);
      if (whole)
        finish<T>(p, s, head0 + c, i - c * dim, sum, joined[c].y);
      else
        mine[i] = sum;
    }
    auto finish_lses = [&]() {
      if (threadIdx.x < cols) finish_lse(p, s, head0 + threadIdx.x, joined[threadIdx.x].x, joined[threadIdx.x].y);
    };
    auto keep_ml = [&](float* piece) {
      if (threadIdx.x < cols) *reinterpret_cast<float2*>(piece + kC * dim + 2 * threadIdx.x) = joined[threadIdx.x];
    };
    // true in the CTA that is the last of `all` to come
    auto last_of = [&](int32_t* counter, int64_t all) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        order = atomicAdd(counter, 1);
        if (order == all - 1) *counter = 0;  // for the next launch
      }
      __syncthreads();
      const bool last = order == all - 1;
      if (last) __threadfence();
      return last;
    };
    // Joins `all` pieces, piece i at piece(i): their sums go to put(c, d, sum).
    auto join = [&](int all, auto piece, auto put) {
      float2* const parts = reinterpret_cast<float2*>(acc);  // [all][cols]: (factor, l)
      for (int i = threadIdx.x; i < all * cols; i += kThreads)
        parts[i] = __ldcg(reinterpret_cast<const float2*>(piece(i / cols) + kC * dim) + i % cols);
      __syncthreads();
      if (threadIdx.x < cols) {
        float2* const of = parts + threadIdx.x;
        float top = kLowest, sum = 0.f;
        for (int i = 0; i < all; ++i) top = fmaxf(top, of[i * cols].x);
        for (int i = 0; i < all; ++i) {
          const float f = join_factor(of[i * cols], top);
          sum += f * of[i * cols].y;
          of[i * cols].x = f;
        }
        joined[threadIdx.x] = make_float2(top, sum);
      }
      __syncthreads();
      // 8 pieces' words at a time: they come from L2, one latency for all
      auto sum_up = [&](auto word) {
        using W = decltype(word);
        constexpr int kE = sizeof(W) / 4;
        for (int i = threadIdx.x * kE; i < cols * dim; i += kThreads * kE) {
          const int c = i / dim;
          float sum[kE] = {};
          for (int k0 = 0; k0 < all; k0 += 8) {
            W o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = __ldcg(reinterpret_cast<const W*>(piece(min(k0 + k, all - 1)) + i));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float f = k0 + k < all ? parts[(k0 + k) * cols + c].x : 0.f;
#pragma unroll
              for (int j = 0; j < kE; ++j)
                if (f != 0.f) sum[j] = fmaf(f, reinterpret_cast<const float*>(&o[k])[j], sum[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < kE; ++j) put(c, i + j - c * dim, sum[j]);
        }
      };
      if (dim % 4 == 0)
        sum_up(float4{});
      else
        sum_up(float{});
    };
    if (whole) {
      finish_lses();
    } else {
      auto put = [&](int c, int d, float sum) { finish<T>(p, s, head0 + c, d, sum, joined[c].y); };
      const int64_t first = c0 + (blockIdx.x - c0) / kFan * kFan;  // of this piece's twenty
      const int64_t near = min(static_cast<int64_t>(kFan), c1 + 1 - first), all = (c1 - c0) / kFan + 1;
      keep_ml(mine);
      if (last_of(p.arrived + 2 * first + (first == c0 ? 1 : 0), near)) {
        auto piece = [&](int i) { return slot(first + i); };
        if (all == 1) {
          join(static_cast<int>(near), piece, put);
          finish_lses();
        } else {
          float* const to = slot(first);
          join(static_cast<int>(near), piece, [&](int c, int d, float sum) { to[c * dim + d] = sum; });
          keep_ml(to);
          if (last_of(p.arrived + 2ll * gridDim.x + c0, all)) {
            join(static_cast<int>(all), [&](int i) { return slot(c0 + i * kFan); }, put);
            finish_lses();
          }
        }
      }
    }
    __syncthreads();
    x += n;
    rest += n;
  }
}

// ── host ───────────────────────────────────────────────────────────────────
struct Kernel {
  void (*attend)(AttendParams) = nullptr;
  int cols = 0;  // query heads per pair
  int ctas = 0;  // per SM
  const char* name = "";
};

template <class Eng>
Kernel kernel_of(const char* name) {
  return {k_attend<Eng>, Eng::kCols, Eng::kCtas, name};
}

template <typename T, int kD>
Kernel mma_kernel(int dim, int group) {
  // More than 8 heads: 16 columns read the keys once (8,000 positions of 16 rows,
  // 16 heads of 128 in bf16, 114 us), two pairs of 8 twice (180).  16 heads of 256
  // dimensions do not fit the registers: two pairs of 8.  A head dim that fills the
  // form has one without bounds on its words: 258 us against 354 at 256, 105
  // against 111 at 64, 77 against 97 at 96.
  if constexpr (kD < 256)
    if (group > 8)
      return dim == kD ? kernel_of<MmaEngine<T, kD, 2, true>>("mma x16") : kernel_of<MmaEngine<T, kD, 2, false>>("mma x16");
  return dim == kD ? kernel_of<MmaEngine<T, kD, 1, true>>("mma x8") : kernel_of<MmaEngine<T, kD, 1, false>>("mma x8");
}

template <typename T>
Kernel mma_kernel(int dim, int group) {
  return dim <= 64    ? mma_kernel<T, 64>(dim, group)
         : dim <= 96  ? mma_kernel<T, 96>(dim, group)
         : dim <= 128 ? mma_kernel<T, 128>(dim, group)
                      : mma_kernel<T, 256>(dim, group);
}

// The widest word that the head dim and the addresses allow, at most 16
// bytes and at most 4 elements, and no more lanes than a row fills.
template <typename T, int kH>
Kernel simt_kernel(int dim, int elements) {
  if (elements >= 4 && dim % 4 == 0) {
    if (dim <= 64) return kernel_of<SimtEngine<T, 4, 1, 16, kH>>("simt 64");
    if (dim <= 128) return kernel_of<SimtEngine<T, 4, 1, 32, kH>>("simt 128");
    return kernel_of<SimtEngine<T, 4, 2, 32, kH>>("simt 256");
  }
  return kernel_of<SimtEngine<T, 1, 8, 32, kH>>("simt");
}

// Columns by the group: a smaller form has fewer sums per lane and more CTAs an SM
// (32 bits; 2 columns against 8: head dim 64 with a window 32 against 53 us, 80 362
// against 496, one head of 128 317 against 427; 4 against 8: 420 against 428).
template <typename T>
Kernel simt_kernel(int dim, int group, int elements) {
  return group <= 2   ? simt_kernel<T, 2>(dim, elements)
         : group <= 4 ? simt_kernel<T, 4>(dim, elements)
                      : simt_kernel<T, 8>(dim, elements);
}

// `align`: the power of two that divides every address and stride, in bytes.
Kernel choose(int32_t dtype, int dim, int group, int align) {
  const int elements = align / akv_dtype_bytes(dtype);
  // 16-bit rows of whole 16-byte words go to the tensor cores: head dim 80 in bf16,
  // 4 query heads, 166 us against 824 for the 32-bit form.
  if (dtype == AKV_F32) return simt_kernel<float>(dim, group, elements);
  if (align >= 16) return dtype == AKV_F16 ? mma_kernel<__half>(dim, group) : mma_kernel<__nv_bfloat16>(dim, group);
  return dtype == AKV_F16 ? simt_kernel<__half>(dim, group, elements) : simt_kernel<__nv_bfloat16>(dim, group, elements);
}

constexpr int kMaxDim = 256;
constexpr int64_t kMaxTokens = 1ll << 30;  // per row: positions are 32-bit numbers

int parts_of(const Kernel& k, int group) { return akv_ceil_div(group, k.cols); }
// Grid of a launch over `rows` rows of at most `chunks` chunks each.
int64_t grid_of(const Kernel& k, int64_t rows, int64_t pairs, int64_t chunks) {
  const int64_t most = rows * pairs * chunks, fit = static_cast<int64_t>(kAkvSMs) * k.ctas;
  static_assert(kAkvSMs * 4 <= kMaxCtas && 3 * kAkvSMs * 4 <= AKV_ATTENTION_COUNTERS, "two levels of joining");
  return most < 1 ? 1 : (most < fit ? most : fit);
}

int64_t chunks_of(int32_t block_size, int32_t width, int32_t keep) {
  const int64_t blocks = keep > 0 && keep < width ? keep : width;
  return (blocks * block_size + kChunk - 1) / kChunk;
}

int64_t scratch_of(const Kernel& k, int64_t grid, int dim) { return grid * 2 * piece_floats(k.cols, dim) * 4; }

// The warps' sums; joining takes their place for a (factor, l) per piece and column.
size_t shared_of(const Kernel& k, int dim) {
  const int sums = kWarps * k.cols * dim * 4, join = 2 * kFan * k.cols * 8;
  return static_cast<size_t>(sums > join ? sums : join);  // at most 32 KiB
}

int power_of_two_in(uint64_t bits) {
  const uint64_t low = bits & (~bits + 1);
  return low == 0 || low > 16 ? 16 : static_cast<int>(low);
}

}  // namespace

int akv_layer_view(const char* what, const AkvPagedPool* p, AkvLayer* out) {
  AKV_ARG_CHECK(p && p->total_blocks > 0 && p->num_layers > 0 && p->num_kv_heads > 0 && p->head_dim > 0,
                "%s: bad pool geometry", what);
  AKV_ARG_CHECK(p->block_size > 0 && (p->block_size & (p->block_size - 1)) == 0,
                "%s: block_size must be a positive power of 2, got %d", what, p->block_size);
  AKV_ARG_CHECK(p->head_dim <= kMaxDim, "%s: head_dim %d is above %d", what, p->head_dim, kMaxDim);
  AKV_ARG_CHECK(p->layer >= 0 && p->layer < p->num_layers, "%s: layer %d of %d", what, p->layer, p->num_layers);
  const int es = akv_dtype_bytes(p->dtype);
  AKV_ARG_CHECK(es > 0, "%s: dtype %d", what, p->dtype);
  AKV_ARG_CHECK(akv_aligned(p->data, es), "%s: pool address not aligned to its type", what);
  out->row_bytes = p->head_dim * es;
  out->tile_bytes = static_cast<int64_t>(p->block_size) * out->row_bytes;
  out->kv_bytes = out->tile_bytes * p->num_kv_heads;
  out->page_bytes = out->kv_bytes * 2 * p->num_layers;
  out->base = static_cast<char*>(p->data) + out->kv_bytes * 2 * p->layer;
  out->total = p->total_blocks;
  out->heads = p->num_kv_heads;
  out->dim = p->head_dim;
  out->bs_log2 = __builtin_ctz(p->block_size);
  return AKV_OK;
}

int akv_tables_view(const char* what, const AkvPageBatch* b, int32_t block_size, AkvTables* out) {
  AKV_ARG_CHECK(b && b->rows >= 0 && b->table_width >= 0 && b->table_stride >= 0, "%s: bad batch", what);
  AKV_ARG_CHECK(static_cast<int64_t>(b->table_width) * block_size <= kMaxTokens, "%s: a table of %d blocks of %d", what,
                b->table_width, block_size);
  AKV_ARG_CHECK(b->rows == 0 || (b->lengths && (b->tables || b->table_width == 0)), "%s: NULL tables or lengths", what);
  out->ids = b->tables;
  out->stride = b->table_stride;
  out->lengths = b->lengths;
  out->width = b->table_width;
  out->rows = b->rows;
  return AKV_OK;
}

int akv_attend_prepare() {
  for (int32_t dtype : {AKV_F32, AKV_F16, AKV_BF16})
    for (int group : {1, 4, 8, 9})
      for (int dim : {56, 64, 80, 96, 104, 128, 200, 256})
        for (int align : {4, 8, 16}) {
          const Kernel k = choose(dtype, dim, group, align);
          if (int rc = akv_load_kernel(reinterpret_cast<const void*>(k.attend), k.name)) return rc;
        }
  return AKV_OK;
}

extern "C" int64_t akv_paged_attention_scratch_bytes(const AkvPagedPool* pool, int32_t rows, int32_t table_width,
                                                     int32_t group, int32_t keep) {
  AkvLayer kv;
  if (akv_layer_view("akv_paged_attention_scratch_bytes", pool, &kv) != AKV_OK) return -1;
  if (rows < 0 || table_width < 0 || group <= 0 || keep < 0) {
    akv_set_error("akv_paged_attention_scratch_bytes: bad arguments");
    return -1;
  }
  const int64_t chunks = chunks_of(pool->block_size, table_width, keep);
  if (rows == 0) return 0;
  int64_t most = 0;
  for (int align : {4, 8, 16}) {  // whichever engine the addresses will allow
    const Kernel k = choose(pool->dtype, kv.dim, group, align);
    const int64_t pairs = static_cast<int64_t>(kv.heads) * parts_of(k, group);
    const int64_t n = scratch_of(k, grid_of(k, rows, pairs, chunks), kv.dim);
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int akv_paged_attention(const AkvPagedPool* pool, const AkvPageBatch* batch, const AkvHeads* query,
                                   int32_t group, float scale, int32_t window, const int32_t* selected, int32_t keep,
                                   const AkvHeads* out, float* lse, void* scratch, int64_t scratch_bytes,
                                   int32_t* counters, AkvStatus* status, void* stream) {
  const char* what = "akv_paged_attention";
  AttendParams p;
  if (int rc = akv_layer_view(what, pool, &p.kv)) return rc;
  if (int rc = akv_tables_view(what, batch, pool->block_size, &p.tab)) return rc;
  if (p.tab.rows == 0) return AKV_OK;
  AKV_ARG_CHECK(pool->data && query && query->data && out && out->data, "%s: NULL pointer", what);
  AKV_ARG_CHECK(group > 0, "%s: group=%d", what, group);
  AKV_ARG_CHECK(static_cast<int64_t>(group) * p.kv.heads <= INT_MAX, "%s: too many query heads", what);
  AKV_ARG_CHECK(window >= 0, "%s: window=%d", what, window);
  AKV_ARG_CHECK(selected == nullptr || keep > 0, "%s: keep=%d", what, keep);
  AKV_ARG_CHECK(query->stride_token >= 0 && query->stride_head >= 0 && out->stride_token >= 0 && out->stride_head >= 0,
                "%s: negative stride", what);
  const int es = akv_dtype_bytes(pool->dtype);
  AKV_ARG_CHECK(akv_aligned(query->data, es) && akv_aligned(out->data, es) && akv_aligned(lse, 4) &&
                    akv_aligned(scratch, 16) && akv_aligned(counters, 4),
                "%s: misaligned pointer", what);
  const uint64_t bits = reinterpret_cast<uintptr_t>(pool->data) | reinterpret_cast<uintptr_t>(query->data) |
                        static_cast<uint64_t>(p.kv.row_bytes) | static_cast<uint64_t>(query->stride_token * es) |
                        static_cast<uint64_t>(query->stride_head * es);
  const Kernel k = choose(pool->dtype, p.kv.dim, group, power_of_two_in(bits));
  p.selected = selected;
  p.keep = selected ? keep : 0;
  p.q = query->data;
  p.q_row = query->stride_token;
  p.q_head = query->stride_head;
  p.out = out->data;
  p.out_row = out->stride_token;
  p.out_head = out->stride_head;
  p.lse = lse;
  p.group = group;
  p.parts = parts_of(k, group);
  p.scale_log2 = scale * kLog2e;
  p.window = window;
  p.st = status;
  const int64_t grid = grid_of(k, p.tab.rows, static_cast<int64_t>(p.kv.heads) * p.parts,
                               chunks_of(pool->block_size, p.tab.width, p.keep));
  const int64_t need = scratch_of(k, grid, p.kv.dim);
  AKV_ARG_CHECK(scratch && scratch_bytes >= need, "%s: scratch has %lld bytes, %lld are needed", what,
                static_cast<long long>(scratch_bytes), static_cast<long long>(need));
  AKV_ARG_CHECK(counters, "%s: NULL counters", what);
  p.pieces = static_cast<float*>(scratch);
  p.arrived = counters;
  k.attend<<<static_cast<unsigned>(grid), kThreads, shared_of(k, p.kv.dim), akv_stream(stream)>>>(p);
  AKV_LAUNCH_CHECK(what);
  return AKV_OK;
}
