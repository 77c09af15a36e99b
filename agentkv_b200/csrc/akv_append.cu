// akv_append.cu — new tokens' keys and values into the paged pool, rotated on
// the way, and the bounds of the blocks that get them.
//
// Rotation: pair (x, y) of a token at position p becomes
// (x cos a - y sin a, y cos a + x sin a), a = p * frequency of the pair; the
// cosines and sines come from a table made once in 64 bits (an angle at
// position 10^5 has lost 5 digits in 32 bits).  Products and sums in 32 bits,
// rounded once to the pool's type.
//
// What bounds it: bytes moved (each operand row read and written once), and
// for a decode step's few rows the launch and two dependent loads.
//
// Work: one unit per (row, block) that gets tokens, dealt to one or several
// CTAs by words of kV elements (with the word of their partners); the four
// lanes that hold a key's word bring its bounds together: no atomics, and the
// same result in any order.  Measured: 8,466 prompt tokens with 32 query and 8 key
// heads of 128 in bf16 66 us (215 MB, 3.3 TB/s; the search, the table and the
// loads come one after the other in a CTA, and 1.8 rounds of CTAs hide little of
// it); replayed from a graph, 256 rows of one token 12.5 us, one row 5.1 us.
#include <climits>

#include "akv_paged.cuh"

namespace {

constexpr int kThreads = 256;
// Query heads that a thread turns together with one load of the angles.  4 with two
// CTAs an SM take 66 us for the prompts (16-byte words of 16-bit types spill 24 bytes a
// thread), 2 with three CTAs took 98.
constexpr int kHeads = 4;

AKV_DEV int32_t akv_ceil_div_dev(int32_t a, int32_t b) { return (a + b - 1) / b; }

struct AppendParams {
  AkvLayer kv;
  AkvTables tab;
  const int32_t* starts;
  int32_t n_tokens;
  const char *key, *value, *query;
  char* query_out;
  int64_t k_tok, k_head, v_tok, v_head, q_tok, q_head, o_tok, o_head;  // strides in bytes
  int32_t q_heads;
  const float* rope;
  int32_t rope_rows, rotary, interleaved;
  char* bounds;
  int64_t bounds_page, bounds_layer;  // bytes
  AkvStatus* st;
};

// New tokens of row s, and how many blocks they fall into.
AKV_DEV int32_t new_tokens(const AppendParams& p, int32_t s) {
  if (p.starts == nullptr) return p.tab.lengths[s] > 0 ? 1 : 0;
  const int32_t from = p.starts[s], to = p.starts[s + 1];
  return from >= 0 && to <= p.n_tokens && to > from ? to - from : 0;
}

AKV_DEV int64_t blocks_touched(const AppendParams& p, int32_t s) {
  const int32_t n = new_tokens(p, s), len = p.tab.lengths[s];
  if (n == 0 || len < n) return 0;
  const int bl = p.kv.bs_log2;
  return ((len - 1) >> bl) - ((len - n) >> bl) + 1;
}

// Whether a pair's two elements lie in different words.
AKV_DEV bool partners(const AppendParams& p, int elements) { return p.rope && (!p.interleaved || elements == 1); }

// One word of a head: dimensions a .. a + kV - 1 and, where they are rotated
// with other words, those of b.
template <typename T, int kV>
struct Lane {
  int a, b;   // b < 0: one word only
  int pair;   // first pair of the word in the table, -1: not rotated

  AKV_DEV void set(const AppendParams& p, int w) {
    const int half = p.rotary / 2;
    const bool apart = partners(p, kV);
    if (apart && w < half / kV) {
      a = p.interleaved ? 2 * w : w * kV;
      b = p.interleaved ? a + 1 : a + half;
      pair = w * kV;
      return;
    }
    if (apart) w += half / kV;  // behind the pairs' two words
    a = w * kV;
    b = -1;
    pair = p.rope && a < p.rotary ? a / 2 : -1;
  }
};

template <typename T, int kV>
AKV_DEV AkvPack<T, kV> word_at(const char* row, int d) {
  return akv_load<T, kV>(row + d * sizeof(T));
}
template <typename T, int kV>
AKV_DEV void load_word(float (&x)[kV], const char* row, int d) {
  akv_unpack<T, kV>(x, word_at<T, kV>(row, d));
}

// Rounds x to T (x holds the rounded values afterwards) and stores it.
template <typename T, int kV>
AKV_DEV void store_word(float (&x)[kV], char* row, int d) {
  *reinterpret_cast<AkvPack<T, kV>*>(row + d * sizeof(T)) = akv_pack<T, kV>(x);
}

// The cosines and sines of a word's pairs at one position.
template <int kV>
struct Turn {
  float cos[kV], sin[kV];  // kV / 2 of each where the word holds whole pairs
};

template <typename T, int kV>
AKV_DEV Turn<kV> load_turn(const AppendParams& p, const Lane<T, kV>& ln, int32_t pos) {
  Turn<kV> t = {};
  if (ln.pair < 0) return t;
  const float* cos_row = p.rope + static_cast<int64_t>(pos) * p.rotary + ln.pair;
  const float* sin_row = cos_row + p.rotary / 2;
  // (words divide the rotary dimensions: their places in the table are as aligned)
  constexpr int kStep = kV >= 8 ? 4 : kV, kHalf = kV > 1 ? kV / 2 : 1;
  if (ln.b >= 0) {
#pragma unroll
    for (int i = 0; i < kV; i += kStep) {
      float c[kStep], n[kStep];
      akv_unpack<float, kStep>(c, akv_load<float, kStep>(cos_row + i));
      akv_unpack<float, kStep>(n, akv_load<float, kStep>(sin_row + i));
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        t.cos[i + j] = c[j];
        t.sin[i + j] = n[j];
      }
    }
  } else if (kV > 1) {
    float c[kHalf], n[kHalf];
    akv_unpack<float, kHalf>(c, akv_load<float, kHalf>(cos_row));
    akv_unpack<float, kHalf>(n, akv_load<float, kHalf>(sin_row));
#pragma unroll
    for (int j = 0; j < kHalf; ++j) {
      t.cos[j] = c[j];
      t.sin[j] = n[j];
    }
  }
  return t;
}

// Turns the word(s) x, y of one token.
template <typename T, int kV>
AKV_DEV void turn(const Turn<kV>& t, const Lane<T, kV>& ln, float (&x)[kV], float (&y)[kV]) {
  if (ln.pair < 0) return;
  if (ln.b >= 0) {
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const float u = x[i], v = y[i];
      x[i] = u * t.cos[i] - v * t.sin[i];
      y[i] = v * t.cos[i] + u * t.sin[i];
    }
  } else if (kV > 1) {
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) {
      const float u = x[2 * i], v = x[(2 * i + 1) % kV];
      x[2 * i] = u * t.cos[i] - v * t.sin[i];
      x[(2 * i + 1) % kV] = v * t.cos[i] + u * t.sin[i];
    }
  }
}

template <typename T, int kV>
AKV_DEV void rotate(const AppendParams& p, const Lane<T, kV>& ln, int32_t pos, float (&x)[kV], float (&y)[kV]) {
  turn(load_turn(p, ln, pos), ln, x, y);
}

template <typename T, int kV>
__global__ void __launch_bounds__(kThreads, 2) k_append(AppendParams p) {
  using Search = AkvRowSearch<kThreads>;
  __shared__ typename Search::Shared sh;
  // One thread reads the record for all: CTAs of this launch write to it while
  // others start, and a CTA whose warps saw different contents would search its
  // row with the sums of warps that have left.
  if (__syncthreads_or(threadIdx.x == 0 && akv_failed(p.st))) return;
  const int bl = p.kv.bs_log2;
  int32_t s;
  int64_t rest = 0;
  if (p.starts == nullptr) {
    s = blockIdx.x;
    if (threadIdx.x == 0 && blockIdx.y == 0 && p.tab.lengths[s] < 0)
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, p.tab.lengths[s], 1);
    if (new_tokens(p, s) == 0) return;
  } else {
    if (blockIdx.y == 0)
      for (int32_t r = blockIdx.x * kThreads + threadIdx.x; r < p.tab.rows; r += gridDim.x * kThreads) {
        const int32_t from = p.starts[r], to = p.starts[r + 1];
        if (from < 0 || to < from || to > p.n_tokens || p.tab.lengths[r] < to - from)
          akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, r, p.tab.lengths[r], to - from);
      }
    auto units = [&](int32_t r) { return blocks_touched(p, r); };
    Search search;
    search.scan(sh, p.tab.rows, units);
    if (blockIdx.x >= search.total) return;
    search.find(sh, blockIdx.x, units, s, rest);
    // (lengths or starts that are written to under the call can leave no such unit)
    if (s < 0 || s >= p.tab.rows || rest < 0 || rest >= blocks_touched(p, s)) return;
  }
  const int32_t len = p.tab.lengths[s], n = new_tokens(p, s), old = len - n;
  const int32_t block = (old >> bl) + static_cast<int32_t>(rest);
  const int64_t from = static_cast<int64_t>(block) << bl, to = from + (1 << bl);
  const int32_t p0 = old > from ? old : static_cast<int32_t>(from);
  const int32_t p1 = len < to ? len : static_cast<int32_t>(to);
  // the first token's row in the operands
  const int64_t row0 = (p.starts ? p.starts[s] : s) + static_cast<int64_t>(p0 - old);
  const int32_t id = block < p.tab.width ? p.tab.ids[s * p.tab.stride + block] : -1;
  const bool placed = static_cast<uint32_t>(id) < static_cast<uint32_t>(p.kv.total);
  const bool turned = p.rope == nullptr || p1 <= p.rope_rows;
  if (!placed || !turned) {
    if (threadIdx.x == 0 && blockIdx.y == 0)
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, placed ? p1 - 1 : id, placed ? p.rope_rows : p.kv.total);
    return;
  }
  const int32_t in0 = static_cast<int32_t>(p0 - from), count = p1 - p0;
  char* page = p.kv.base + id * p.kv.page_bytes;
  // words of a head: a rotated one with its partner counts once
  const int all = p.kv.dim / kV;
  const int words = partners(p, kV) ? all - p.rotary / 2 / kV : all;
  const int32_t heads = p.kv.heads;
  // Items: a word of a key through every fourth token, four lanes next to one
  // another for the four (they bring its bounds together); a word of a value,
  // likewise; a word of one token of four query heads, which turn alike.
  const int64_t keys = 4ll * heads * words, values = 4ll * heads * all;
  const int64_t items = keys + values + static_cast<int64_t>(akv_ceil_div_dev(p.q_heads, kHeads)) * count * words;
  for (int64_t it = blockIdx.y * kThreads + threadIdx.x; it < items; it += static_cast<int64_t>(gridDim.y) * kThreads) {
    if (it < keys) {
      const int q = static_cast<int>(it & 3);
      const int32_t h = static_cast<int32_t>((it >> 2) / words);
      Lane<T, kV> ln;
      ln.set(p, static_cast<int>((it >> 2) % words));
      char* tile = page + h * p.kv.tile_bytes;
      float lo[kV], hi[kV], lo2[kV], hi2[kV];
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        lo[i] = lo2[i] = INFINITY;
        hi[i] = hi2[i] = -INFINITY;
      }
      auto take = [&](const float(&x)[kV], const float(&y)[kV]) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          lo[i] = min_nan(lo[i], x[i]);
          hi[i] = max_nan(hi[i], x[i]);
          lo2[i] = min_nan(lo2[i], y[i]);
          hi2[i] = max_nan(hi2[i], y[i]);
        }
      };
      if (p.bounds)
#pragma unroll 4
        for (int32_t r = q; r < in0; r += 4) {
          float x[kV], y[kV] = {};
          load_word<T, kV>(x, tile + static_cast<int64_t>(r) * p.kv.row_bytes, ln.a);
          if (ln.b >= 0) load_word<T, kV>(y, tile + static_cast<int64_t>(r) * p.kv.row_bytes, ln.b);
          take(x, y);
        }
#pragma unroll 4
      for (int32_t t = q; t < count; t += 4) {
        const char* src = p.key + (row0 + t) * p.k_tok + h * p.k_head;
        char* dst = tile + static_cast<int64_t>(in0 + t) * p.kv.row_bytes;
        float x[kV], y[kV] = {};
        load_word<T, kV>(x, src, ln.a);
        if (ln.b >= 0) load_word<T, kV>(y, src, ln.b);
        rotate<T, kV>(p, ln, p0 + t, x, y);
        store_word<T, kV>(x, dst, ln.a);
        if (ln.b >= 0) store_word<T, kV>(y, dst, ln.b);
        take(x, y);
      }
      if (p.bounds) {
        const uint32_t four = 0xfu << (threadIdx.x & 28);
#pragma unroll
        for (int off = 1; off < 4; off <<= 1)
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            lo[i] = min_nan(lo[i], __shfl_xor_sync(four, lo[i], off));
            hi[i] = max_nan(hi[i], __shfl_xor_sync(four, hi[i], off));
            lo2[i] = min_nan(lo2[i], __shfl_xor_sync(four, lo2[i], off));
            hi2[i] = max_nan(hi2[i], __shfl_xor_sync(four, hi2[i], off));
          }
        char* b = p.bounds + id * p.bounds_page + p.bounds_layer + static_cast<int64_t>(h) * 2 * p.kv.row_bytes;
        if (q == 0) store_word<T, kV>(lo, b, ln.a);
        if (q == 1) store_word<T, kV>(hi, b + p.kv.row_bytes, ln.a);
        if (ln.b >= 0) {
          if (q == 2) store_word<T, kV>(lo2, b, ln.b);
          if (q == 3) store_word<T, kV>(hi2, b + p.kv.row_bytes, ln.b);
        }
      }
    } else if (it < keys + values) {  // a value: bits only
      const int64_t i = (it - keys) / all;
      const int q = static_cast<int>(i & 3);
      const int32_t h = static_cast<int32_t>(i >> 2);
      const int d = static_cast<int>((it - keys) % all) * kV * static_cast<int>(sizeof(T));
      const char* src = p.value + row0 * p.v_tok + h * p.v_head + d;
      char* dst = page + p.kv.kv_bytes + h * p.kv.tile_bytes + static_cast<int64_t>(in0) * p.kv.row_bytes + d;
#pragma unroll 4
      for (int32_t t = q; t < count; t += 4)
        *reinterpret_cast<AkvPack<T, kV>*>(dst + static_cast<int64_t>(t) * p.kv.row_bytes) =
            akv_load<T, kV>(src + t * p.v_tok);
    } else {  // queries
      const int64_t i = (it - keys - values) / words;
      const int32_t t = static_cast<int32_t>(i % count), h0 = static_cast<int32_t>(i / count) * kHeads;
      Lane<T, kV> ln;
      ln.set(p, static_cast<int>((it - keys - values) % words));
      const Turn<kV> by = load_turn(p, ln, p0 + t);
      const char* src = p.query + (row0 + t) * p.q_tok + h0 * p.q_head;
      char* dst = p.query_out + (row0 + t) * p.o_tok + h0 * p.o_head;
      AkvPack<T, kV> a[kHeads], b[kHeads];
#pragma unroll
      for (int k = 0; k < kHeads; ++k)
        if (h0 + k < p.q_heads) {
          a[k] = word_at<T, kV>(src + k * p.q_head, ln.a);
          if (ln.b >= 0) b[k] = word_at<T, kV>(src + k * p.q_head, ln.b);
        }
#pragma unroll
      for (int k = 0; k < kHeads; ++k)
        if (h0 + k < p.q_heads) {
          float x[kV], y[kV] = {};
          akv_unpack<T, kV>(x, a[k]);
          if (ln.b >= 0) akv_unpack<T, kV>(y, b[k]);
          turn(by, ln, x, y);
          store_word<T, kV>(x, dst + k * p.o_head, ln.a);
          if (ln.b >= 0) store_word<T, kV>(y, dst + k * p.o_head, ln.b);
        }
    }
  }
}

// The bounds of every block of every row, from its keys: one warp per (row,
// block, head), a lane per element.  41,783 blocks of 16 keys, 8 heads of 128 in
// bf16: 497 us, 3.1 TB/s (one element per lane and load: a load brings 64 bytes).
template <typename T>
__global__ void __launch_bounds__(kThreads) k_bounds(AppendParams p) {
  if (akv_failed(p.st)) return;
  const int lane = threadIdx.x & 31, bl = p.kv.bs_log2;
  const int64_t per_row = static_cast<int64_t>(p.tab.width) * p.kv.heads;
  const int64_t items = p.tab.rows * per_row;
  for (int64_t it = blockIdx.x * (kThreads / 32ll) + threadIdx.x / 32; it < items; it += gridDim.x * (kThreads / 32ll)) {
    const int32_t s = static_cast<int32_t>(it / per_row);
    const int32_t block = static_cast<int32_t>(it % per_row / p.kv.heads), h = static_cast<int32_t>(it % p.kv.heads);
    const int32_t len = akv_held(p.tab, bl, s);
    if (block == 0 && h == 0 && lane == 0 && p.tab.lengths[s] != len)
      akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, p.tab.lengths[s], p.tab.width);
    const int64_t from = static_cast<int64_t>(block) << bl;
    if (from >= len) continue;
    const int32_t rows = static_cast<int32_t>(len - from < (1 << bl) ? len - from : (1 << bl));
    const int32_t id = p.tab.ids[s * p.tab.stride + block];
    if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.kv.total)) {
      if (h == 0 && lane == 0) akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, id, p.kv.total);
      continue;
    }
    const char* tile = p.kv.base + id * p.kv.page_bytes + h * p.kv.tile_bytes;
    char* b = p.bounds + id * p.bounds_page + p.bounds_layer + static_cast<int64_t>(h) * 2 * p.kv.row_bytes;
    for (int d = lane; d < p.kv.dim; d += 32) {
      float lo = INFINITY, hi = -INFINITY;
#pragma unroll 8
      for (int32_t r = 0; r < rows; ++r) {
        const float x = to_f32<T>(reinterpret_cast<const T*>(tile + static_cast<int64_t>(r) * p.kv.row_bytes)[d]);
        lo = min_nan(lo, x);
        hi = max_nan(hi, x);
      }
      reinterpret_cast<T*>(b)[d] = from_f32<T>(lo);
      reinterpret_cast<T*>(b + p.kv.row_bytes)[d] = from_f32<T>(hi);
    }
  }
}

using AppendKernel = void (*)(AppendParams);

// `elements`: the largest word, in elements, that every address, stride and
// the rotary half allow.
template <typename T>
AppendKernel append_kernel(int elements) {
  if constexpr (sizeof(T) == 2)
    if (elements >= 8) return k_append<T, 8>;
  if (elements >= 4) return k_append<T, 4>;
  if (elements >= 2) return k_append<T, 2>;
  return k_append<T, 1>;
}

AppendKernel append_kernel(int32_t dtype, int elements) {
  return dtype == AKV_F32 ? append_kernel<float>(elements)
                          : dtype == AKV_F16 ? append_kernel<__half>(elements) : append_kernel<__nv_bfloat16>(elements);
}

AppendKernel bounds_kernel(int32_t dtype) {
  return dtype == AKV_F32 ? k_bounds<float> : dtype == AKV_F16 ? k_bounds<__half> : k_bounds<__nv_bfloat16>;
}

int lowest_bit(uint64_t bits) { return static_cast<int>(bits & (~bits + 1) & 31); }

}  // namespace

int akv_append_prepare() {
  for (int32_t dtype : {AKV_F32, AKV_F16, AKV_BF16}) {
    for (int n : {1, 2, 4, 8})
      if (int rc = akv_load_kernel(reinterpret_cast<const void*>(append_kernel(dtype, n)), "akv_prepare: k_append"))
        return rc;
    if (int rc = akv_load_kernel(reinterpret_cast<const void*>(bounds_kernel(dtype)), "akv_prepare: k_bounds"))
      return rc;
  }
  return AKV_OK;
}

extern "C" int akv_kv_append(const AkvPagedPool* pool, const AkvPageBatch* batch, const AkvHeads* key,
                             const AkvHeads* value, int32_t n_tokens, const int32_t* starts, const float* rope,
                             int32_t rope_rows, int32_t rotary_dim, int32_t interleaved, const AkvHeads* query,
                             const AkvHeads* query_out, int32_t n_query_heads, void* bounds, AkvStatus* status,
                             void* stream) {
  const char* what = "akv_kv_append";
  AppendParams p = {};
  if (int rc = akv_layer_view(what, pool, &p.kv)) return rc;
  if (int rc = akv_tables_view(what, batch, pool->block_size, &p.tab)) return rc;
  AKV_ARG_CHECK(n_tokens >= 0, "%s: n_tokens=%d", what, n_tokens);
  AKV_ARG_CHECK(starts || n_tokens == p.tab.rows, "%s: %d tokens for %d rows of one token each", what, n_tokens,
                p.tab.rows);
  if (n_tokens == 0 || p.tab.rows == 0) return AKV_OK;
  AKV_ARG_CHECK(pool->data && key && key->data && value && value->data, "%s: NULL pointer", what);
  AKV_ARG_CHECK(n_query_heads >= 0 && (n_query_heads == 0 || (query && query->data && query_out && query_out->data)),
                "%s: bad query", what);
  AKV_ARG_CHECK(rope == nullptr || (rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= p.kv.dim && rope_rows >= 0),
                "%s: rotary_dim=%d of head_dim %d, %d rows", what, rotary_dim, p.kv.dim, rope_rows);
  const int es = akv_dtype_bytes(pool->dtype);
  uint64_t bits = reinterpret_cast<uintptr_t>(pool->data) | static_cast<uint64_t>(p.kv.row_bytes) |
                  reinterpret_cast<uintptr_t>(bounds);
  for (const AkvHeads* x : {key, value, n_query_heads ? query : key, n_query_heads ? query_out : key}) {
    AKV_ARG_CHECK(x->stride_token >= 0 && x->stride_head >= 0, "%s: negative stride", what);
    AKV_ARG_CHECK(akv_aligned(x->data, es), "%s: misaligned pointer", what);
    bits |= reinterpret_cast<uintptr_t>(x->data) | static_cast<uint64_t>(x->stride_token * es) |
            static_cast<uint64_t>(x->stride_head * es);
  }
  AKV_ARG_CHECK(akv_aligned(rope, 16) && akv_aligned(bounds, es), "%s: misaligned pointer", what);
  // a word lies wholly in one half of the rotated pairs, or holds whole pairs
  if (rope) bits |= static_cast<uint64_t>(interleaved ? rotary_dim : rotary_dim / 2) * es;
  const int low = lowest_bit(bits);
  const int elements = (low == 0 || low > 16 ? 16 : low) / es;
  p.starts = starts;
  p.n_tokens = n_tokens;
  p.key = static_cast<const char*>(key->data);
  p.k_tok = key->stride_token * es;
  p.k_head = key->stride_head * es;
  p.value = static_cast<const char*>(value->data);
  p.v_tok = value->stride_token * es;
  p.v_head = value->stride_head * es;
  p.q_heads = n_query_heads;
  if (n_query_heads) {
    p.query = static_cast<const char*>(query->data);
    p.q_tok = query->stride_token * es;
    p.q_head = query->stride_head * es;
    p.query_out = static_cast<char*>(query_out->data);
    p.o_tok = query_out->stride_token * es;
    p.o_head = query_out->stride_head * es;
  }
  p.rope = rope;
  p.rope_rows = rope_rows;
  p.rotary = rope ? rotary_dim : 0;
  p.interleaved = interleaved != 0;
  p.bounds = static_cast<char*>(bounds);
  p.bounds_layer = static_cast<int64_t>(p.kv.heads) * 2 * p.kv.row_bytes * pool->layer;
  p.bounds_page = static_cast<int64_t>(p.kv.heads) * 2 * p.kv.row_bytes * pool->num_layers;
  p.st = status;
  // a row's n tokens lie in at most n, and at most n / block_size + 2, blocks
  const int64_t most = n_tokens / pool->block_size + 2ll * p.tab.rows;
  const int64_t units = starts == nullptr ? p.tab.rows : most < n_tokens ? most : n_tokens;
  // As many CTAs per unit as its words fill, while all are resident (2 an SM):
  // a CTA has four latencies behind it (its row, its block, then words) before
  // the first word moves, so waves of them cost more than a longer loop.
  const int64_t words = p.kv.dim / elements;
  const int64_t items = words * (8ll * p.kv.heads + (starts ? 4ll : 1ll) * p.q_heads / kHeads);
  int64_t per = (items + kThreads - 1) / kThreads;
  const int64_t room = 2ll * kAkvSMs / units;
  per = per < room ? per : room;
  const dim3 grid(static_cast<unsigned>(units), static_cast<unsigned>(per < 1 ? 1 : per > 65535 ? 65535 : per));
  append_kernel(pool->dtype, elements)<<<grid, kThreads, 0, akv_stream(stream)>>>(p);
  AKV_LAUNCH_CHECK(what);
  return AKV_OK;
}

extern "C" int akv_key_bounds(const AkvPagedPool* pool, const AkvPageBatch* batch, void* bounds, AkvStatus* status,
                              void* stream) {
  const char* what = "akv_key_bounds";
  AppendParams p = {};
  if (int rc = akv_layer_view(what, pool, &p.kv)) return rc;
  if (int rc = akv_tables_view(what, batch, pool->block_size, &p.tab)) return rc;
  if (p.tab.rows == 0 || p.tab.width == 0) return AKV_OK;
  AKV_ARG_CHECK(pool->data && bounds, "%s: NULL pointer", what);
  AKV_ARG_CHECK(akv_aligned(bounds, akv_dtype_bytes(pool->dtype)), "%s: misaligned pointer", what);
  p.bounds = static_cast<char*>(bounds);
  p.bounds_layer = static_cast<int64_t>(p.kv.heads) * 2 * p.kv.row_bytes * pool->layer;
  p.bounds_page = static_cast<int64_t>(p.kv.heads) * 2 * p.kv.row_bytes * pool->num_layers;
  p.st = status;
  const int64_t warps = static_cast<int64_t>(p.tab.rows) * p.tab.width * p.kv.heads;
  const int64_t ctas = (warps + kThreads / 32 - 1) / (kThreads / 32), most = 16ll * kAkvSMs;
  bounds_kernel(pool->dtype)<<<static_cast<unsigned>(ctas < most ? ctas : most), kThreads, 0, akv_stream(stream)>>>(p);
  AKV_LAUNCH_CHECK(what);
  return AKV_OK;
}
