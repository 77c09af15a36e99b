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
// Work: (row, key head, up to kHeads query heads) pairs of chunks of 64
// positions.  All chunks of the batch, in that order, are dealt to the CTAs in
// equal contiguous ranges, whatever the rows' lengths are (the host does not know
// them, and a captured launch replays with others): a pair that lies inside
// one range is finished there, one that crosses ranges leaves a piece in
// scratch per CTA, and k_join joins them.
#include <climits>

#include "akv_paged.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 16;               // positions per warp and step
constexpr int kChunk = kTile * kWarps;  // positions per CTA and step
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A running maximum is raised only once a score lies this far above it (the
// sums are the same for any m, so long as 2^(x - m) stays in range: at most
// 2^8 here), which spares most steps the reduction over the lanes.
constexpr float kLazy = 8.0f;

struct AttendMeta {
  int32_t row, head, part, pieces;
};

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
  int32_t direct;  // one CTA per pair, nothing to join
  float* pieces;
  AttendMeta* meta;
  AkvStatus* st;
};

// Row s: positions [lo, n) take part; its pairs have chunks [first, first + chunks).
struct Extent {
  int32_t n, lo, first, chunks;
};

AKV_DEV Extent row_extent(const AttendParams& p, int32_t s) {
  Extent e;
  e.n = akv_held(p.tab, p.kv.bs_log2, s);
  e.lo = p.window > 0 && e.n > p.window ? e.n - p.window : 0;
  if (p.selected) {
    const int64_t blocks = (static_cast<int64_t>(e.n) + (1 << p.kv.bs_log2) - 1) >> p.kv.bs_log2;
    const int64_t taken = (blocks < p.keep ? blocks : p.keep) << p.kv.bs_log2;
    e.first = 0;
    e.chunks = static_cast<int32_t>((taken + kChunk - 1) / kChunk);
  } else {
    e.first = e.lo / kChunk;
    e.chunks = static_cast<int32_t>((static_cast<int64_t>(e.n) + kChunk - 1) / kChunk) - e.first;
  }
  return e;
}

// A warp's view of the blocks under its tiles: lane i holds one table entry,
// for the next 32 (or fewer, where a tile spans several blocks) tiles.
struct Cursor {
  int32_t id, place;  // this lane's block (-1: none) and its place in the table
  int32_t from;       // the first chunk that the entries are for

  AKV_DEV static int entries(int bs_log2) { return bs_log2 >= 4 ? 1 : 16 >> bs_log2; }

  AKV_DEV void refill(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t chunk, int32_t end,
                      int warp, int lane) {
    from = chunk;
    const int bl = p.kv.bs_log2, per = entries(bl);
    const int64_t c = static_cast<int64_t>(chunk) + lane / per;
    const int64_t tok = c * kChunk + warp * kTile + (static_cast<int64_t>(lane % per) << bl);
    const int64_t vb = tok >> bl;
    const int64_t blocks = (static_cast<int64_t>(e.n) + (1 << bl) - 1) >> bl;
    id = -1;
    place = -1;
    if (c >= end) return;
    if (p.selected) {
      if (vb >= p.keep || vb >= blocks) return;
      place = p.selected[(static_cast<int64_t>(s) * p.kv.heads + h) * p.keep + vb];
      if (place < -1 || place >= blocks) {
        akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, place, static_cast<int32_t>(blocks));
        place = -1;
      }
      if (place < 0 || ((static_cast<int64_t>(place) + 1) << bl) <= e.lo) return;
    } else {
      if (vb >= blocks || ((vb + 1) << bl) <= e.lo) return;
      place = static_cast<int32_t>(vb);
    }
    id = p.tab.ids[s * p.tab.stride + place];
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.kv.total)) {
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, id, p.kv.total);
      id = -1;
    }
  }
  // The lane that holds the entry of position r (0..15) of chunk's tile.
  AKV_DEV int lane_of(int bs_log2, int32_t chunk, int r) const {
    return (chunk - from) * entries(bs_log2) + (bs_log2 >= 4 ? 0 : r >> bs_log2);
  }
  AKV_DEV bool covers(int bs_log2, int32_t chunk) const { return (chunk - from + 1) * entries(bs_log2) <= 32; }

  // Which of the tile's 16 positions take part (bit r), and the tile's first
  // position within its block (its rows lie behind one another there).
  AKV_DEV uint32_t valid(const AttendParams& p, const Extent& e, int32_t chunk, int warp, int lane) const {
    const int bl = p.kv.bs_log2, r = lane & 15;
    const int src = lane_of(bl, chunk, r);
    const int32_t b = __shfl_sync(kFullWarp, id, src);
    const int32_t at = __shfl_sync(kFullWarp, place, src);
    const int32_t in = (chunk * kChunk + warp * kTile + r) & ((1 << bl) - 1);
    const int64_t pos = (static_cast<int64_t>(at) << bl) + in;
    const bool ok = b >= 0 && pos >= e.lo && pos < e.n;
    return __ballot_sync(kFullWarp, ok) & 0xffffu;
  }
};

// ── tensor-core engine: 16-bit types, head dims 64, 96, 128, 256 ────────────
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
// 2 c + 1, 2 c + 8, 2 c + 9).  The next tile's keys are loaded as soon as this one's have been
// used, this one's values while the scores are computed.
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

AKV_DEV uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

AKV_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Streaming loads: a block is read once per launch.
AKV_DEV uint4 ld16(const char* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
AKV_DEV uint2 ld8(const char* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }

template <typename T, int kD, int kN>
struct MmaEngine {
  using Type = T;
  static constexpr int kDim = kD;          // compiled for this head dim
  static constexpr int kHeads = 8 * kN;    // query heads per pair
  static constexpr int kCtas = kD <= 128 && kN == 1 ? 3 : (kD <= 128 ? 2 : 1);
  static constexpr int kKi = kD / 32;      // 16-byte words of a key row per lane
  static constexpr int kVi = kD / 64;      // the same of a value row,
  static constexpr bool kVr = kD % 64 != 0;  // and 8 bytes more
  static constexpr int kMt = kD / 16;      // output tiles of 16 dimensions

  uint4 q[kN][kKi];
  uint4 ka[kKi], kb[kKi];
  uint4 v[4][kVi > 0 ? kVi : 1];
  uint2 vr[4];
  float o[kN][kMt][4];
  float m[kN][2], l[kN][2];

  AKV_DEV void load_k(const AttendParams& p, const Cursor& cur, const char* kbase, int32_t chunk, uint32_t vm, int warp,
                      int lane) {
    const int g = lane >> 2, c = lane & 3, bl = p.kv.bs_log2;
    const int32_t ida = __shfl_sync(kFullWarp, cur.id, cur.lane_of(bl, chunk, g));
    const int32_t idb = __shfl_sync(kFullWarp, cur.id, cur.lane_of(bl, chunk, g + 8));
    const int32_t t0 = chunk * kChunk + warp * kTile, mask = (1 << bl) - 1;
    const char* pa = kbase + ida * p.kv.page_bytes + ((t0 + g) & mask) * (kD * 2) + c * 16;
    const char* pb = kbase + idb * p.kv.page_bytes + ((t0 + g + 8) & mask) * (kD * 2) + c * 16;
    if (vm == 0xffffu) {
#pragma unroll
      for (int i = 0; i < kKi; ++i) {
        ka[i] = ld16(pa + i * 64);
        kb[i] = ld16(pb + i * 64);
      }
    } else {
      const bool va = (vm >> g) & 1, vb = (vm >> (g + 8)) & 1;
#pragma unroll
      for (int i = 0; i < kKi; ++i) {
        ka[i] = va ? ld16(pa + i * 64) : make_uint4(0, 0, 0, 0);
        kb[i] = vb ? ld16(pb + i * 64) : make_uint4(0, 0, 0, 0);
      }
    }
  }

  // Values of positions that take no part are 0, whatever the block holds.
  AKV_DEV void load_v(const AttendParams& p, const Cursor& cur, const char* vbase, int32_t chunk, uint32_t vm, int warp,
                      int lane) {
    const int g = lane >> 2, c = lane & 3, bl = p.kv.bs_log2;
    const int32_t t0 = chunk * kChunk + warp * kTile, mask = (1 << bl) - 1;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int r = 2 * c + (x & 1) + (x >> 1) * 8;
      const int32_t id = __shfl_sync(kFullWarp, cur.id, cur.lane_of(bl, chunk, r));
      const char* pv = vbase + id * p.kv.page_bytes + ((t0 + r) & mask) * (kD * 2);
      if (vm == 0xffffu || ((vm >> r) & 1)) {
#pragma unroll
        for (int i = 0; i < kVi; ++i) v[x][i] = ld16(pv + i * 128 + g * 16);
        if (kVr) vr[x] = ld8(pv + kVi * 128 + g * 8);
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
    for (int n = 0; n < kN; ++n) {
      Pack2<T>::mma(o[n][tile], a0, a1, a2, a3, hi[n][0], hi[n][1]);
      Pack2<T>::mma(o[n][tile], a0, a1, a2, a3, lo[n][0], lo[n][1]);
    }
  }

  // Chunks [a, b) of pair (s, h, part).
  AKV_DEV void run(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t part, int32_t a, int32_t b,
                   int warp, int lane) {
    const int g = lane >> 2, c = lane & 3;
    const char* kbase = p.kv.base + h * p.kv.tile_bytes;
    const char* vbase = kbase + p.kv.kv_bytes;
    Cursor cur;
    cur.refill(p, e, s, h, a, b, warp, lane);
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int32_t head = part * kHeads + n * 8 + g;
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + head) * p.q_head;
#pragma unroll
      for (int i = 0; i < kKi; ++i)
        q[n][i] = head < p.group ? ld16(reinterpret_cast<const char*>(row + i * 32 + c * 8)) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int t = 0; t < kMt; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][t][x] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    uint32_t vm = cur.valid(p, e, a, warp, lane);
    load_k(p, cur, kbase, a, vm, warp, lane);
    for (int32_t chunk = a; chunk < b; ++chunk) {
      load_v(p, cur, vbase, chunk, vm, warp, lane);
      float sc[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < kKi; ++i) {
          Pack2<T>::mma(sc[n], ka[i].x, kb[i].x, ka[i].y, kb[i].y, q[n][i].x, q[n][i].y);
          Pack2<T>::mma(sc[n], ka[i].z, kb[i].z, ka[i].w, kb[i].w, q[n][i].z, q[n][i].w);
        }
      }
      const uint32_t now = vm;
      if (chunk + 1 < b) {
        if (!cur.covers(p.kv.bs_log2, chunk + 1)) cur.refill(p, e, s, h, chunk + 1, b, warp, lane);
        vm = cur.valid(p, e, chunk + 1, warp, lane);
        load_k(p, cur, kbase, chunk + 1, vm, warp, lane);
      }
      bool raise = false;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sc[n][x] *= p.scale_log2;
          if (!((now >> (g + (x >> 1) * 8)) & 1)) sc[n][x] = -INFINITY;
        }
        raise |= fmaxf(sc[n][0], sc[n][2]) > m[n][0] + kLazy;
        raise |= fmaxf(sc[n][1], sc[n][3]) > m[n][1] + kLazy;
      }
      if (__any_sync(kFullWarp, raise)) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(sc[n][x], sc[n][x + 2]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, off));
            const float to = fmaxf(m[n][x], top);
            const float by = to == -INFINITY ? 1.f : exp2_fast(m[n][x] - to);
            m[n][x] = to;
            l[n][x] *= by;
#pragma unroll
            for (int t = 0; t < kMt; ++t) {
              o[n][t][x] *= by;
              o[n][t][x + 2] *= by;
            }
          }
      }
      // The weights go into the product as the sum of two 16-bit numbers:
      // one alone would be off by half a step of the type, as much as the
      // output's own rounding; the time is the memory's either way.
      uint32_t hi[kN][2], lo[kN][2];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float w0 = exp2_fast(sc[n][2 * x] - m0), w1 = exp2_fast(sc[n][2 * x + 1] - m1);
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

  // This warp's sums: acc [kHeads][kD], and m and l of each head.
  AKV_DEV void store(float* acc, float2* ml, int /*dim*/, int lane) {
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
          *reinterpret_cast<float2*>(acc + head * kD + d) = make_float2(o[n][t][x], o[n][t][x + 2]);
        }
      }
  }
};

// ── 32-bit engine: any type and head dim (up to 256) ───────────────────────
// Multiplies and adds in 32 bits.  A lane holds kE consecutive dimensions of
// every 32 kE; 4 positions at a time give 4 * kHeads partial scores per lane,
// which halving exchanges turn into one whole score (or a copy) per lane.
template <typename T, int kE, int kJ, int kH>
struct SimtEngine {
  using Type = T;
  static constexpr int kDim = 0;
  static constexpr int kHeads = kH;
  static constexpr int kCtas = kH * kE * kJ >= 64 ? 2 : 3;
  static constexpr int kX = kE * kJ;       // dimensions per lane
  static constexpr int kU = 4;             // positions at a time
  static constexpr int kVals = kU * kH;    // scores at a time,
  static constexpr int kStep = 32 / kVals;  // each held by this many lanes
  using Vec = AkvVec<T, kE>;

  float q[kH][kX], o[kH][kX];
  float m, l;  // of this lane's head, l over this lane's position of each four

  AKV_DEV static void load_row(float (&x)[kX], const char* row, int dim, bool ok, int lane) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int d = (j * 32 + lane) * kE;
      if (ok && d < dim) {
        const Vec w = *reinterpret_cast<const Vec*>(row + d * sizeof(T));
#pragma unroll
        for (int i = 0; i < kE; ++i) x[j * kE + i] = to_f32<T>(w.v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) x[j * kE + i] = 0.f;
      }
    }
  }

  AKV_DEV void run(const AttendParams& p, const Extent& e, int32_t s, int32_t h, int32_t part, int32_t a, int32_t b,
                   int warp, int lane) {
    const char* kbase = p.kv.base + h * p.kv.tile_bytes;
    const char* vbase = kbase + p.kv.kv_bytes;
    const int bl = p.kv.bs_log2, mask = (1 << bl) - 1;
    Cursor cur;
    cur.refill(p, e, s, h, a, b, warp, lane);
#pragma unroll
    for (int n = 0; n < kH; ++n) {
      const int32_t head = part * kH + n;
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + head) * p.q_head;
      load_row(q[n], reinterpret_cast<const char*>(row), p.kv.dim, head < p.group, lane);
#pragma unroll
      for (int x = 0; x < kX; ++x) o[n][x] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    const int mine = lane / kStep % kU;  // this lane's position of each four
    for (int32_t chunk = a; chunk < b; ++chunk) {
      if (!cur.covers(bl, chunk)) cur.refill(p, e, s, h, chunk, b, warp, lane);
      const uint32_t vm = cur.valid(p, e, chunk, warp, lane);
      if (vm == 0) continue;
      const int32_t t0 = chunk * kChunk + warp * kTile;
#pragma unroll 1
      for (int r0 = 0; r0 < kTile; r0 += kU) {
        float k[kU][kX], v[kU][kX];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int r = r0 + u;
          const int32_t id = __shfl_sync(kFullWarp, cur.id, cur.lane_of(bl, chunk, r));
          const int64_t off = id * p.kv.page_bytes + static_cast<int64_t>((t0 + r) & mask) * p.kv.row_bytes;
          load_row(k[u], kbase + off, p.kv.dim, (vm >> r) & 1, lane);
          load_row(v[u], vbase + off, p.kv.dim, (vm >> r) & 1, lane);
        }
        float val[kVals];
#pragma unroll
        for (int n = 0; n < kH; ++n)
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            float d = 0.f;
#pragma unroll
            for (int x = 0; x < kX; ++x) d = fmaf(q[n][x], k[u][x], d);
            val[n * kU + u] = d;
          }
        // value i ends, whole, in lanes i * kStep ..: each exchange keeps
        // the half of the values that belongs to this lane's half
        int off = 16;
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
        const bool in = (vm >> (r0 + mine)) & 1;
        const float sc = in ? val[0] * p.scale_log2 : -INFINITY;
        if (__any_sync(kFullWarp, sc > m + kLazy)) {
          float top = sc;
          top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, kStep));
          top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, 2 * kStep));
          const float to = fmaxf(m, top);
          const float by = to == -INFINITY ? 1.f : exp2f(m - to);
          m = to;
          l *= by;
#pragma unroll
          for (int n = 0; n < kH; ++n) {
            const float f = __shfl_sync(kFullWarp, by, n * kU * kStep);
#pragma unroll
            for (int x = 0; x < kX; ++x) o[n][x] *= f;
          }
        }
        const float w = exp2f(sc - (m == -INFINITY ? 0.f : m));
        l += w;
#pragma unroll
        for (int n = 0; n < kH; ++n)
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            const float f = __shfl_sync(kFullWarp, w, (n * kU + u) * kStep);
#pragma unroll
            for (int x = 0; x < kX; ++x) o[n][x] = fmaf(f, v[u][x], o[n][x]);
          }
      }
    }
  }

  AKV_DEV void store(float* acc, float2* ml, int dim, int lane) {
    float sum = l;
    sum += __shfl_xor_sync(kFullWarp, sum, kStep);
    sum += __shfl_xor_sync(kFullWarp, sum, 2 * kStep);
    if (lane % (kU * kStep) == 0) ml[lane / (kU * kStep)] = make_float2(m, sum);
#pragma unroll
    for (int n = 0; n < kH; ++n)
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          const int d = (j * 32 + lane) * kE + i;
          if (d < dim) acc[n * dim + d] = o[n][j * kE + i];
        }
  }
};

// The factor that brings sums taken with maximum m to maximum `to` (both may be -inf: no sums).
AKV_DEV float join_factor(float m, float to) { return m == -INFINITY ? 0.f : exp2f(m - to); }

template <typename T>
AKV_DEV void finish(const AttendParams& p, int32_t s, int32_t head, int d, float o, float l) {
  T* out = static_cast<T*>(p.out) + s * p.out_row + head * p.out_head;
  out[d] = from_f32<T>(l == 0.f ? 0.f : o / l);
}

AKV_DEV void finish_lse(const AttendParams& p, int32_t s, int32_t head, float m, float l) {
  if (p.lse)
    p.lse[static_cast<int64_t>(s) * p.kv.heads * p.group + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

AKV_HD int64_t piece_floats(int heads, int dim) { return static_cast<int64_t>(heads) * (dim + 2); }

template <class Eng>
__global__ void __launch_bounds__(kThreads, Eng::kCtas) k_attend(AttendParams p) {
  using T = typename Eng::Type;
  constexpr int kH = Eng::kHeads;
  using Search = AkvRowSearch<kThreads>;
  extern __shared__ __align__(16) float acc[];  // [kWarps][kH][dim]
  __shared__ float2 ml[kWarps][kH];
  __shared__ float factor[kWarps][kH];
  __shared__ float2 joined[kH];
  __shared__ typename Search::Shared sh;
  akv_grid_release();  // k_join may take its place; it waits for this grid's end
  if (akv_failed(p.st)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dim = Eng::kDim ? Eng::kDim : p.kv.dim;
  const int64_t pairs = static_cast<int64_t>(p.kv.heads) * p.parts;  // of a row
  auto units = [&](int32_t s) -> int64_t { return row_extent(p, s).chunks * pairs; };

  int32_t s = 0;
  int64_t rest = 0, x = 0, end = 0, total = 0, ctas = gridDim.x;
  AttendMeta meta = {0, 0, 0, 0};
  if (p.direct) {
    s = static_cast<int32_t>(blockIdx.x / pairs);
    const int32_t chunks = row_extent(p, s).chunks;
    rest = blockIdx.x % pairs * chunks;
    end = chunks;
  } else {
    Search search;
    search.scan(sh, p.tab.rows, units);
    total = search.total;
    if (ctas > total) ctas = total;
    if (blockIdx.x < ctas) {
      x = total * blockIdx.x / ctas;
      end = total * (blockIdx.x + 1) / ctas;
      search.find(sh, x, units, s, rest);
    }
  }
  // rows that hold nothing, and lengths that the table cannot hold
  for (int32_t r = blockIdx.x; r < p.tab.rows; r += gridDim.x) {
    if (threadIdx.x == 0 && p.tab.lengths[r] > akv_held(p.tab, p.kv.bs_log2, r))
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, r, p.tab.lengths[r], p.tab.width);
    if (row_extent(p, r).chunks == 0) {
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
    {
      Eng eng;
      eng.run(p, e, s, h, part, e.first + a, e.first + a + n, warp, lane);
      eng.store(acc + warp * kH * dim, ml[warp], dim, lane);
    }
    __syncthreads();
    if (threadIdx.x < kH) {
      const int i = threadIdx.x;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w][i].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        factor[w][i] = join_factor(ml[w][i].x, top);
        sum += factor[w][i] * ml[w][i].y;
      }
      joined[i] = make_float2(top, sum);
    }
    __syncthreads();
    const bool whole = a == 0 && n == e.chunks;
    const int32_t left = p.group - part * kH;
    const int heads = left < kH ? left : kH;
    float* piece = nullptr;
    if (!whole) {
      // a pair that begins here and goes on is the CTA's second piece
      piece = p.pieces + (blockIdx.x * 2ll + (a == 0 ? 1 : 0)) * piece_floats(kH, dim);
      if (a == 0) {
        const int64_t stop = x + e.chunks;
        int64_t last = (stop * ctas + total - 1) / total - 1;
        while (total * (last + 1) / ctas < stop) ++last;
        while (last > blockIdx.x && total * last / ctas >= stop) --last;
        meta = AttendMeta{s, h, part, static_cast<int32_t>(last - blockIdx.x)};
      }
    }
    for (int i = threadIdx.x; i < heads * dim; i += kThreads) {
      const int head = i / dim, d = i - head * dim;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        sum += factor[w][head] == 0.f ? 0.f : factor[w][head] * acc[(w * kH + head) * dim + d];
      if (whole)
        finish<T>(p, s, h * p.group + part * kH + head, d, sum, joined[head].y);
      else
        piece[i] = sum;
    }
    if (threadIdx.x < heads) {
      const float2 j = joined[threadIdx.x];
      if (whole)
        finish_lse(p, s, h * p.group + part * kH + threadIdx.x, j.x, j.y);
      else
        *reinterpret_cast<float2*>(piece + kH * dim + 2 * threadIdx.x) = j;
    }
    __syncthreads();
    x += n;
    rest += n;
  }
  if (!p.direct && threadIdx.x == 0) p.meta[blockIdx.x] = meta;
}

// Joins the pieces of the pair that began in CTA blockIdx.x and went on:
// that CTA's second piece and the first pieces of the CTAs behind it.
// `split` warps share a head's pieces, 8 / split heads per CTA.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) k_join(AttendParams p, int32_t heads_per_pair, int32_t split) {
  constexpr int kX = 8;  // dimensions per lane: head dims up to 256
  __shared__ float sums[kJoinThreads / 32][kX * 32];
  akv_grid_wait();
  if (akv_failed(p.st)) return;
  const AttendMeta meta = p.meta[blockIdx.x];
  if (meta.pieces <= 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = p.kv.dim;
  const int head = blockIdx.y * (kJoinThreads / 32 / split) + warp / split, sub = warp % split;
  const int32_t left = p.group - meta.part * heads_per_pair;
  const bool live = head < heads_per_pair && head < left;
  const int64_t size = piece_floats(heads_per_pair, dim);
  const int n = meta.pieces + 1;
  auto slot = [&](int i) -> const float* {
    return p.pieces + (i == 0 ? blockIdx.x * 2ll + 1 : (static_cast<int64_t>(blockIdx.x) + i) * 2) * size;
  };
  float m = -INFINITY, l = 0.f, o[kX];
#pragma unroll
  for (int x = 0; x < kX; ++x) o[x] = 0.f;
  if (live) {
    for (int i = lane; i < n; i += 32) m = fmaxf(m, slot(i)[heads_per_pair * dim + 2 * head]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullWarp, m, off));
    for (int i = lane; i < n; i += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(slot(i) + heads_per_pair * dim + 2 * head);
      l += join_factor(ml.x, m) * ml.y;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(kFullWarp, l, off);
#pragma unroll 2
    for (int i = sub; i < n; i += split) {
      const float* at = slot(i);
      const float f = join_factor(at[heads_per_pair * dim + 2 * head], m);
      if (f == 0.f) continue;
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        const int d = x * 32 + lane;
        if (d < dim) o[x] = fmaf(f, at[head * dim + d], o[x]);
      }
    }
  }
  if (split > 1) {
#pragma unroll
    for (int x = 0; x < kX; ++x) sums[warp][x * 32 + lane] = o[x];
    __syncthreads();
    if (sub == 0)
      for (int w = 1; w < split; ++w)
#pragma unroll
        for (int x = 0; x < kX; ++x) o[x] += sums[warp + w][x * 32 + lane];
  }
  if (live && sub == 0) {
    const int32_t qh = meta.head * p.group + meta.part * heads_per_pair + head;
#pragma unroll
    for (int x = 0; x < kX; ++x) {
      const int d = x * 32 + lane;
      if (d < dim) finish<T>(p, meta.row, qh, d, o[x], l);
    }
    if (lane == 0) finish_lse(p, meta.row, qh, m, l);
  }
}

// ── host ───────────────────────────────────────────────────────────────────
struct Kernel {
  void (*attend)(AttendParams) = nullptr;
  void (*join)(AttendParams, int32_t, int32_t) = nullptr;
  int heads = 0;  // query heads per pair
  int ctas = 0;   // per SM
  const char* name = "";
};

template <class Eng>
Kernel kernel_of(const char* name) {
  return {k_attend<Eng>, k_join<typename Eng::Type>, Eng::kHeads, Eng::kCtas, name};
}

template <typename T>
Kernel mma_kernel(int dim, int group) {
  const bool wide = group > 8;
  switch (dim) {
    case 64: return wide ? kernel_of<MmaEngine<T, 64, 2>>("mma 64x16") : kernel_of<MmaEngine<T, 64, 1>>("mma 64x8");
    case 96: return wide ? kernel_of<MmaEngine<T, 96, 2>>("mma 96x16") : kernel_of<MmaEngine<T, 96, 1>>("mma 96x8");
    case 128: return wide ? kernel_of<MmaEngine<T, 128, 2>>("mma 128x16") : kernel_of<MmaEngine<T, 128, 1>>("mma 128x8");
    // 16 heads of 256 dimensions do not fit the registers: two pairs of 8
    case 256: return kernel_of<MmaEngine<T, 256, 1>>("mma 256x8");
    default: return {};
  }
}

// The widest word that the head dim and the addresses allow, at most 16
// bytes and at most 4 elements.
template <typename T>
Kernel simt_kernel(int dim, int group, int elements) {
  const bool wide = group > 2;
  if (elements >= 4 && dim % 4 == 0 && dim > 64)
    return wide ? kernel_of<SimtEngine<T, 4, 2, 8>>("simt 4x2x8") : kernel_of<SimtEngine<T, 4, 2, 2>>("simt 4x2x2");
  if (elements >= 2 && dim % 2 == 0)
    return wide ? kernel_of<SimtEngine<T, 2, 4, 8>>("simt 2x4x8") : kernel_of<SimtEngine<T, 2, 4, 2>>("simt 2x4x2");
  return wide ? kernel_of<SimtEngine<T, 1, 8, 8>>("simt 1x8x8") : kernel_of<SimtEngine<T, 1, 8, 2>>("simt 1x8x2");
}

// `align`: the power of two that divides every address and stride, in bytes.
Kernel choose(int32_t dtype, int dim, int group, int align) {
  const int elements = align / akv_dtype_bytes(dtype);
  if (dtype == AKV_F32) return simt_kernel<float>(dim, group, elements);
  Kernel k;
  if (align >= 16) k = dtype == AKV_F16 ? mma_kernel<__half>(dim, group) : mma_kernel<__nv_bfloat16>(dim, group);
  if (k.attend) return k;
  return dtype == AKV_F16 ? simt_kernel<__half>(dim, group, elements) : simt_kernel<__nv_bfloat16>(dim, group, elements);
}

constexpr int kDirectChunks = 4;  // tables of at most so many chunks: one CTA per pair, no joining launch
constexpr int kMaxDim = 256;
constexpr int64_t kMaxTokens = 1ll << 30;  // per row: positions are 32-bit numbers

// Grid of a launch over `rows` rows of at most `chunks` chunks each.
int64_t grid_of(const Kernel& k, int64_t rows, int64_t pairs, int64_t chunks, bool direct) {
  if (direct) return rows * pairs;
  const int64_t most = rows * pairs * chunks, fit = static_cast<int64_t>(kAkvSMs) * k.ctas;
  return most < 1 ? 1 : (most < fit ? most : fit);
}

int64_t chunks_of(int32_t block_size, int32_t width, int32_t keep) {
  const int64_t blocks = keep > 0 && keep < width ? keep : width;
  return (blocks * block_size + kChunk - 1) / kChunk;
}

int64_t scratch_of(const Kernel& k, int64_t grid, int dim) {
  return grid * (2 * piece_floats(k.heads, dim) * 4 + static_cast<int64_t>(sizeof(AttendMeta)));
}

// at most 32 KiB: 16 heads of 128 dimensions, or 8 of 256
size_t shared_of(const Kernel& k, int dim) { return static_cast<size_t>(kWarps) * k.heads * dim * 4; }

int prepare(const Kernel& k) {
  if (int rc = akv_load_kernel(reinterpret_cast<const void*>(k.attend), k.name)) return rc;
  return akv_load_kernel(reinterpret_cast<const void*>(k.join), k.name);
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
    for (int group : {1, 4, 9}) {
      for (int dim : {64, 96, 128, 256})
        if (int rc = prepare(choose(dtype, dim, group, 16))) return rc;
      for (int align : {1, 2, 4, 8, 16})
        if (align >= akv_dtype_bytes(dtype))
          if (int rc = prepare(choose(dtype, 80, group, align))) return rc;
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
  if (rows == 0 || chunks <= kDirectChunks) return 0;
  int64_t most = 0;
  for (int align : {4, 16}) {  // whichever engine the addresses will allow
    const Kernel k = choose(pool->dtype, kv.dim, group, align);
    const int64_t pairs = static_cast<int64_t>(kv.heads) * akv_ceil_div(group, k.heads);
    const int64_t n = scratch_of(k, grid_of(k, rows, pairs, chunks, false), kv.dim);
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int akv_paged_attention(const AkvPagedPool* pool, const AkvPageBatch* batch, const AkvHeads* query,
                                   int32_t group, float scale, int32_t window, const int32_t* selected, int32_t keep,
                                   const AkvHeads* out, float* lse, void* scratch, int64_t scratch_bytes,
                                   AkvStatus* status, void* stream) {
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
                    akv_aligned(scratch, 16),
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
  p.parts = akv_ceil_div(group, k.heads);
  p.scale_log2 = scale * kLog2e;
  p.window = window;
  p.st = status;
  const int64_t pairs = static_cast<int64_t>(p.kv.heads) * p.parts;
  const int64_t chunks = chunks_of(pool->block_size, p.tab.width, p.keep);
  p.direct = chunks <= kDirectChunks;
  const int64_t grid = grid_of(k, p.tab.rows, pairs, chunks, p.direct);
  AKV_ARG_CHECK(grid <= INT_MAX, "%s: too many rows", what);
  const int64_t need = p.direct ? 0 : scratch_of(k, grid, p.kv.dim);
  AKV_ARG_CHECK(scratch_bytes >= need && (scratch || need == 0), "%s: scratch has %lld bytes, %lld are needed", what,
                static_cast<long long>(scratch_bytes), static_cast<long long>(need));
  p.meta = static_cast<AttendMeta*>(scratch);
  p.pieces = reinterpret_cast<float*>(p.meta + (p.direct ? 0 : grid));
  cudaStream_t st = akv_stream(stream);
  k.attend<<<static_cast<unsigned>(grid), kThreads, shared_of(k, p.kv.dim), st>>>(p);
  AKV_LAUNCH_CHECK(what);
  if (p.direct) return AKV_OK;
  // few pairs leave many pieces each: the more warps share a head's
  const int32_t split = static_cast<int64_t>(p.tab.rows) * pairs * 8 <= grid ? 8 : 2;
  const int32_t per = kJoinThreads / 32 / split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), akv_ceil_div(group < k.heads ? group : k.heads, per));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, k.join, p, static_cast<int32_t>(k.heads), split);
  if (err != cudaSuccess) return akv_cuda_fail(err, what);
  return AKV_OK;
}
