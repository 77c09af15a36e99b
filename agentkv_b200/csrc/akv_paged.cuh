// akv_paged.cuh — what the operators over the paged key-value pool share:
// the pool's geometry, element types, the search for a row in a ragged
// batch, and programmatic dependent launch.
#pragma once

#include <cstring>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "akv_common.cuh"

constexpr uint32_t kFullWarp = 0xffffffffu;

template <typename T>
AKV_DEV float to_f32(T x);
template <>
AKV_DEV float to_f32<float>(float x) { return x; }
template <>
AKV_DEV float to_f32<__half>(__half x) { return __half2float(x); }
template <>
AKV_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
AKV_DEV T from_f32(float x);
template <>
AKV_DEV float from_f32<float>(float x) { return x; }
template <>
AKV_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
AKV_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <int kBytes>
struct AkvWord;
template <>
struct AkvWord<16> { using Type = uint4; };
template <>
struct AkvWord<8> { using Type = uint2; };
template <>
struct AkvWord<4> { using Type = uint32_t; };
template <>
struct AkvWord<2> { using Type = uint16_t; };

// `N` elements of T as one word: loaded, held and stored whole (an array of
// 16-bit elements takes a register each), taken apart where they are used.
template <typename T, int N>
using AkvPack = typename AkvWord<static_cast<int>(sizeof(T)) * N>::Type;

template <typename T, int N>
AKV_DEV AkvPack<T, N> akv_load(const void* p) {
  return *static_cast<const AkvPack<T, N>*>(p);
}

template <typename T, int N>
AKV_DEV void akv_unpack(float (&x)[N], const AkvPack<T, N>& w) {
  if constexpr (sizeof(T) == 4) {
    memcpy(x, &w, sizeof(x));
  } else if constexpr (N == 1) {
    T t;
    memcpy(&t, &w, sizeof(t));
    x[0] = to_f32<T>(t);
  } else {
    uint32_t u[N / 2];
    memcpy(u, &w, sizeof(u));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}

// Rounds x to T (x holds the rounded values afterwards).
template <typename T, int N>
AKV_DEV AkvPack<T, N> akv_pack(float (&x)[N]) {
  AkvPack<T, N> w;
  T t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = from_f32<T>(x[i]);
    x[i] = to_f32<T>(t[i]);
  }
  memcpy(&w, t, sizeof(w));
  return w;
}

// min / max that a NaN on either side makes NaN
AKV_DEV float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
AKV_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Waits until the launches before this one in the stream have ended and their
// writes can be seen; a launch without the programmatic attribute passes.
AKV_DEV void akv_grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// One layer of the pool [total][L][2][H][bs][D], in bytes.
struct AkvLayer {
  char* base;          // page 0, this layer, K, head 0
  int64_t page_bytes;  // page b: base + b * page_bytes
  int64_t tile_bytes;  // head h: + h * tile_bytes
  int64_t kv_bytes;    // V: + kv_bytes
  int32_t row_bytes;   // position r: + r * row_bytes
  int32_t total, heads, dim;
  int32_t bs_log2;
};

// The ragged batch's block tables.
struct AkvTables {
  const int32_t* ids;
  int64_t stride;
  const int32_t* lengths;
  int32_t width, rows;
};

// The tokens that row s holds: its length, cut to what its table can hold.
AKV_DEV int32_t akv_held(const AkvTables& t, int32_t bs_log2, int32_t s) {
  const int32_t len = t.lengths[s];
  const int64_t most = static_cast<int64_t>(t.width) << bs_log2;
  return len < 0 ? 0 : static_cast<int32_t>(len < most ? len : most);
}

// Finds the row that holds unit x of a batch whose row s has count(s) units:
// thread t sums the counts of a contiguous stretch of rows, a scan over the
// block gives the stretches' bases, and the thread whose stretch holds x
// walks it.
template <int kThreads>
struct AkvRowSearch {
  static constexpr int kWarps = kThreads / 32;
  struct Shared {
    int64_t warp_sum[kWarps];
    int64_t rest;
    int32_t row;
  };
  int64_t base = 0, sum = 0;  // this thread's stretch
  int64_t total = 0;
  int32_t first = 0, last = 0;

  template <class F>
  AKV_DEV void scan(Shared& sh, int32_t rows, F count) {
    const int32_t per = (rows + kThreads - 1) / kThreads;
    const int64_t from = static_cast<int64_t>(threadIdx.x) * per;
    first = static_cast<int32_t>(from < rows ? from : rows);
    last = static_cast<int32_t>(from + per < rows ? from + per : rows);
    sum = 0;
    for (int32_t s = first; s < last; ++s) sum += count(s);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(kFullWarp, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) sh.warp_sum[warp] = incl;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int64_t ws = sh.warp_sum[w];
      before += w < warp ? ws : 0;
      total += ws;
    }
    base = before + incl - sum;
  }

  // Row and place inside it of unit x < total (all threads, after scan()).
  template <class F>
  AKV_DEV void find(Shared& sh, int64_t x, F count, int32_t& row, int64_t& rest) {
    if (x >= base && x < base + sum) {
      int64_t at = x - base;
      int32_t s = first;
      for (; s + 1 < last; ++s) {
        const int64_t n = count(s);
        if (at < n) break;
        at -= n;
      }
      sh.row = s;
      sh.rest = at;
    }
    __syncthreads();
    row = sh.row;
    rest = sh.rest;
  }
};

// ── host ───────────────────────────────────────────────────────────────────
inline int akv_dtype_bytes(int32_t dtype) {
  return dtype == AKV_F32 ? 4 : (dtype == AKV_F16 || dtype == AKV_BF16) ? 2 : 0;
}

// Checks the pool's geometry; fills the layer's view.
int akv_layer_view(const char* what, const AkvPagedPool* p, AkvLayer* out);
// Checks the batch's tables.
int akv_tables_view(const char* what, const AkvPageBatch* b, int32_t block_size, AkvTables* out);

inline bool akv_aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
