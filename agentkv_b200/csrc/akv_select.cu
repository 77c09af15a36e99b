// akv_select.cu — the blocks of each row that matter most to its new token.
//
// With a block's key bounds kmin <= k <= kmax by dimension, no key of it
// scores above sum_d max(q_d kmin_d, q_d kmax_d).  max(q a, q b) is q b for
// q > 0 and q a for q < 0, so the sum over a group of query heads is
//   sum_d P_d kmax_d + N_d kmin_d,  P_d = sum_heads max(q_d, 0), N_d = sum_heads min(q_d, 0):
// two products per dimension whatever the group.
//
// Scores are held in 64 bits: which of two blocks is taken hangs on the last
// places of their scores, and products of 16-bit numbers and their sums are
// exact there, so the choice does not depend on the order of a sum.
//
// What bounds it: 2 head_dim elements read per block and key head.  (The conversions to 64
// bits come near: 16 a clock and SM, against the 11 or so elements that HBM
// brings in that clock.)
#include <climits>

#include "akv_paged.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kSelectThreads = 512;
constexpr int kTask = 64;          // blocks per warp and task
constexpr int kSharedKeys = 8192;  // keys that k_select holds in shared memory
constexpr double kLargest = 1.7976931348623157e308;

struct SelectParams {
  AkvLayer kv;  // geometry only
  AkvTables tab;
  const char* bounds;
  int64_t bounds_page;  // bytes
  const void* q;
  int64_t q_row, q_head;
  int32_t group, keep, first, last;
  uint64_t* keys;  // [rows][heads][width]
  int32_t* selected;
  AkvStatus* st;
};

AKV_DEV int32_t blocks_of(const SelectParams& p, int32_t s) {
  return static_cast<int32_t>((static_cast<int64_t>(akv_held(p.tab, p.kv.bs_log2, s)) + (1 << p.kv.bs_log2) - 1) >>
                              p.kv.bs_log2);
}

// The score as a whole number of the same order, above 0 and below the
// largest; NaN counts as the highest score.
AKV_DEV uint64_t key_of(double x) {
  x = x != x ? kLargest : fmin(fmax(x, -kLargest), kLargest);
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));  // -0 and 0 are equal
  return u >> 63 ? ~u : u | (1ull << 63);
}

template <typename T, int kE, int kJ>
__global__ void __launch_bounds__(kThreads) k_score(SelectParams p) {
  if (akv_failed(p.st)) return;
  const int lane = threadIdx.x & 31, dim = p.kv.dim;
  const int64_t groups = (p.tab.width + kTask - 1) / kTask;
  const int64_t tasks = p.tab.rows * groups * p.kv.heads;
  const int64_t layer_bytes = 2ll * p.kv.row_bytes;
  for (int64_t t = blockIdx.x * (kThreads / 32ll) + threadIdx.x / 32; t < tasks; t += gridDim.x * (kThreads / 32ll)) {
    const int32_t h = static_cast<int32_t>(t % p.kv.heads);
    const int32_t s = static_cast<int32_t>(t / p.kv.heads / groups);
    const int32_t j0 = static_cast<int32_t>(t / p.kv.heads % groups) * kTask;
    const int32_t n = blocks_of(p, s);
    if (n <= p.keep || j0 >= n) continue;
    double coef[kJ * kE];
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < kE; ++i) coef[j * kE + i] = 0.0;
    for (int32_t g = 0; g < p.group; ++g) {
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + g) * p.q_head;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int at = (j * 32 + lane) * kE;
        if (at < 2 * dim) {
          const bool high = at >= dim;
#pragma unroll
          for (int i = 0; i < kE; ++i) {
            const float q = to_f32<T>(row[(high ? at - dim : at) + i]);
            coef[j * kE + i] += q != q ? static_cast<double>(q) : high ? fmax(q, 0.f) : fmin(q, 0.f);
          }
        }
      }
    }
    const char* base = p.bounds + h * layer_bytes;
    const int32_t stop = n - j0 < kTask ? n - j0 : kTask;
    for (int32_t c0 = 0; c0 < stop; c0 += 32) {
      int32_t id = 0;
      if (c0 + lane < stop) {
        id = p.tab.ids[s * p.tab.stride + j0 + c0 + lane];
        if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.kv.total)) {
          if (h == 0) akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, id, p.kv.total);
          id = 0;
        }
      }
      for (int32_t c = c0; c < c0 + 32 && c < stop; c += 8) {
        double sum[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const char* box = base + __shfl_sync(kFullWarp, id, c - c0 + u) * p.bounds_page;
          sum[u] = 0.0;
          if (c + u < stop) {
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              const int at = (j * 32 + lane) * kE;
              if (at < 2 * dim) {
                const AkvVec<T, kE> w = *reinterpret_cast<const AkvVec<T, kE>*>(box + at * sizeof(T));
#pragma unroll
                for (int i = 0; i < kE; ++i)
                  sum[u] = fma(coef[j * kE + i], static_cast<double>(to_f32<T>(w.v[i])), sum[u]);
              }
            }
          }
        }
        // sum u ends, whole, in lanes 4 u .. 4 u + 3, added in the same order for every u
        int off = 16;
#pragma unroll
        for (int w = 4; w >= 1; w >>= 1, off >>= 1) {
          const bool up = lane & off;
#pragma unroll
          for (int i = 0; i < w; ++i) {
            const double send = up ? sum[i] : sum[i + w], keep = up ? sum[i + w] : sum[i];
            sum[i] = keep + __shfl_xor_sync(kFullWarp, send, off);
          }
        }
        sum[0] += __shfl_xor_sync(kFullWarp, sum[0], 2);
        sum[0] += __shfl_xor_sync(kFullWarp, sum[0], 1);
        const int32_t mine = c + lane / 4;
        if (lane % 4 == 0 && mine < stop)
          p.keys[(static_cast<int64_t>(s) * p.kv.heads + h) * p.tab.width + j0 + mine] = key_of(sum[0]);
      }
    }
  }
}

// One CTA per (row, key head): a radix selection finds the lowest key that is
// taken, digit by digit from the highest bit in which the keys differ, until
// a digit's keys are all taken; then one pass in order writes the places.
__global__ void __launch_bounds__(kSelectThreads) k_select(SelectParams p) {
  extern __shared__ __align__(16) uint64_t held[];
  __shared__ uint64_t ends[2][kSelectThreads / 32];
  __shared__ int32_t bins[256];
  __shared__ int32_t found[2];  // digit, keys above it
  __shared__ uint32_t counts[2][kSelectThreads / 32];
  akv_grid_wait();
  if (akv_failed(p.st)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t s = blockIdx.x / p.kv.heads;
  const int32_t n = blocks_of(p, s);
  int32_t* out = p.selected + static_cast<int64_t>(blockIdx.x) * p.keep;
  if (tid == 0 && blockIdx.x % p.kv.heads == 0 && p.tab.lengths[s] > akv_held(p.tab, p.kv.bs_log2, s))
    akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, p.tab.lengths[s], p.tab.width);
  if (n <= p.keep) {
    for (int32_t i = tid; i < p.keep; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* keys = p.keys + static_cast<int64_t>(blockIdx.x) * p.tab.width;
  const bool local = n <= kSharedKeys;
  const int32_t from = p.first, to = n - p.last;  // [from, to) are ranked
  uint64_t lo = ~0ull, hi = 0;
  for (int32_t j = from + tid; j < to; j += kSelectThreads) {
    const uint64_t k = keys[j];
    if (local) held[j] = k;
    lo = k < lo ? k : lo;
    hi = k > hi ? k : hi;
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    const uint64_t a = __shfl_xor_sync(kFullWarp, lo, off), b = __shfl_xor_sync(kFullWarp, hi, off);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  if (lane == 0) {
    ends[0][warp] = lo;
    ends[1][warp] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    lo = ends[0][w] < lo ? ends[0][w] : lo;
    hi = ends[1][w] > hi ? ends[1][w] : hi;
  }
  auto key = [&](int32_t j) { return local ? held[j] : keys[j]; };
  // keys with (key & mask) == prefix are still in question, `need` of them are taken
  int32_t need = p.keep - p.first - p.last;
  int bit = lo == hi ? 0 : 64 - __clzll(static_cast<long long>(lo ^ hi));  // bits below this differ
  uint64_t mask = bit == 64 ? 0 : ~0ull << bit, prefix = hi & mask;
  while (bit > 0 && need > 0) {
    const int width = bit < 8 ? bit : 8;
    bit -= width;
    if (tid < 256) bins[tid] = 0;
    __syncthreads();
    for (int32_t j = from + tid; j < to; j += kSelectThreads) {
      const uint64_t k = key(j);
      if ((k & mask) == prefix) atomicAdd(&bins[(k >> bit) & ((1 << width) - 1)], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // lane i: digits 255 - 8 i .. 248 - 8 i, highest first
      int32_t sum = 0, at[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        at[i] = bins[255 - 8 * lane - i];
        sum += at[i];
      }
      int32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t up = __shfl_up_sync(kFullWarp, incl, o);
        if (lane >= o) incl += up;
      }
      int32_t above = incl - sum;
      if (above < need && incl >= need) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < need && above + at[i] >= need) {
            found[0] = 255 - 8 * lane - i;
            found[1] = above;
          }
          above += at[i];
        }
      }
    }
    __syncthreads();
    const int32_t digit = found[0], count = bins[digit];
    need -= found[1];
    mask |= static_cast<uint64_t>((1 << width) - 1) << bit;
    prefix |= static_cast<uint64_t>(digit) << bit;
    __syncthreads();
    if (count == need) break;  // all of them
  }
  // taken: keys above the prefix's range, and the first `need` of those in it
  int32_t above = 0, equal = 0;
  int flip = 0;
  for (int32_t j0 = 0; j0 < n; j0 += kSelectThreads, flip ^= 1) {
    const int32_t j = j0 + tid;
    bool gt = false, eq = false;
    if (j < n) {
      if (j < from || j >= to) {
        gt = true;
      } else {
        const uint64_t k = key(j) & mask;
        gt = k > prefix;
        eq = k == prefix;
      }
    }
    const uint32_t bg = __ballot_sync(kFullWarp, gt), be = __ballot_sync(kFullWarp, eq);
    if (lane == 0) counts[flip][warp] = __popc(bg) | (__popc(be) << 16);
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      const uint32_t c = counts[flip][w];
      before += w < warp ? c : 0;
      all += c;
    }
    const uint32_t below = (1u << lane) - 1;
    const int32_t g = above + static_cast<int32_t>(before & 0xffff) + __popc(bg & below);
    const int32_t e = equal + static_cast<int32_t>(before >> 16) + __popc(be & below);
    if (gt || (eq && e < need)) out[g + (e < need ? e : need)] = j;
    above += static_cast<int32_t>(all & 0xffff);
    equal += static_cast<int32_t>(all >> 16);
  }
}

using ScoreKernel = void (*)(SelectParams);

// The widest word that the addresses and the head dim allow; a lane holds
// every 32nd word of a block's bounds.
template <typename T>
ScoreKernel score_kernel(int dim, int elements) {
  constexpr int kWide = 16 / sizeof(T);
  if (elements >= kWide) {
    if (2 * dim <= 32 * kWide) return k_score<T, kWide, 1>;
    if (2 * dim <= 64 * kWide) return k_score<T, kWide, 2>;
    return k_score<T, kWide, sizeof(T) == 4 ? 4 : 2>;
  }
  if (elements >= 2) return k_score<T, 2, 8>;
  return k_score<T, 1, 16>;
}

ScoreKernel score_kernel(int32_t dtype, int dim, int elements) {
  return dtype == AKV_F32 ? score_kernel<float>(dim, elements)
                          : dtype == AKV_F16 ? score_kernel<__half>(dim, elements)
                                             : score_kernel<__nv_bfloat16>(dim, elements);
}

int64_t key_bytes(int64_t rows, int64_t heads, int64_t width, int64_t keep) {
  return width <= keep ? 0 : rows * heads * width * 8;
}

int allow_shared() {
  const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(k_select),
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedKeys * 8);
  return e == cudaSuccess ? AKV_OK : akv_cuda_fail(e, "k_select: shared memory");
}

}  // namespace

int akv_select_prepare() {
  for (int32_t dtype : {AKV_F32, AKV_F16, AKV_BF16})
    for (int dim : {32, 64, 128, 256})
      for (int elements : {1, 2, 8})
        if (int rc = akv_load_kernel(reinterpret_cast<const void*>(score_kernel(dtype, dim, elements)),
                                     "akv_prepare: k_score"))
          return rc;
  if (int rc = akv_load_kernel(reinterpret_cast<const void*>(k_select), "akv_prepare: k_select")) return rc;
  return allow_shared();
}

extern "C" int64_t akv_select_blocks_scratch_bytes(int32_t rows, int32_t num_kv_heads, int32_t table_width,
                                                   int32_t keep) {
  if (rows < 0 || num_kv_heads <= 0 || table_width < 0 || keep <= 0) {
    akv_set_error("akv_select_blocks_scratch_bytes: bad arguments");
    return -1;
  }
  return key_bytes(rows, num_kv_heads, table_width, keep);
}

extern "C" int akv_select_blocks(const AkvPagedPool* pool, const void* bounds, const AkvPageBatch* batch,
                                 const AkvHeads* query, int32_t group, int32_t keep, int32_t first, int32_t last,
                                 int32_t* selected, void* scratch, int64_t scratch_bytes, AkvStatus* status,
                                 void* stream) {
  const char* what = "akv_select_blocks";
  SelectParams p = {};
  if (int rc = akv_layer_view(what, pool, &p.kv)) return rc;
  if (int rc = akv_tables_view(what, batch, pool->block_size, &p.tab)) return rc;
  AKV_ARG_CHECK(group > 0 && keep > 0 && first >= 0 && last >= 0 && static_cast<int64_t>(first) + last <= keep,
                "%s: group=%d keep=%d first=%d last=%d", what, group, keep, first, last);
  if (p.tab.rows == 0) return AKV_OK;
  AKV_ARG_CHECK(bounds && query && query->data && selected, "%s: NULL pointer", what);
  AKV_ARG_CHECK(query->stride_token >= 0 && query->stride_head >= 0, "%s: negative stride", what);
  const int es = akv_dtype_bytes(pool->dtype);
  AKV_ARG_CHECK(akv_aligned(bounds, es) && akv_aligned(query->data, es) && akv_aligned(selected, 4) &&
                    akv_aligned(scratch, 16),
                "%s: misaligned pointer", what);
  const int64_t need = key_bytes(p.tab.rows, p.kv.heads, p.tab.width, keep);
  AKV_ARG_CHECK(scratch_bytes >= need && (scratch || need == 0), "%s: scratch has %lld bytes, %lld are needed", what,
                static_cast<long long>(scratch_bytes), static_cast<long long>(need));
  const int64_t pairs = static_cast<int64_t>(p.tab.rows) * p.kv.heads;
  AKV_ARG_CHECK(pairs <= INT_MAX, "%s: too many rows", what);
  const int64_t head_bytes = 2ll * p.kv.row_bytes, layer_bytes = head_bytes * p.kv.heads;
  p.bounds = static_cast<const char*>(bounds) + layer_bytes * pool->layer;
  p.bounds_page = layer_bytes * pool->num_layers;
  p.q = query->data;
  p.q_row = query->stride_token;
  p.q_head = query->stride_head;
  p.group = group;
  p.keep = keep;
  p.first = first;
  p.last = last;
  p.keys = static_cast<uint64_t*>(scratch);
  p.selected = selected;
  p.st = status;
  cudaStream_t st = akv_stream(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs));
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  if (need) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(bounds) | static_cast<uint64_t>(p.kv.row_bytes);
    const int low = static_cast<int>(bits & (~bits + 1) & 31);
    const int64_t warps = pairs * ((p.tab.width + kTask - 1) / kTask), per = kThreads / 32;
    const int64_t ctas = (warps + per - 1) / per, most = 8ll * kAkvSMs;
    score_kernel(pool->dtype, p.kv.dim, (low == 0 || low > 16 ? 16 : low) / es)<<<
        static_cast<unsigned>(ctas < most ? ctas : most), kThreads, 0, st>>>(p);
    AKV_LAUNCH_CHECK(what);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.tab.width < kSharedKeys ? p.tab.width : kSharedKeys) * 8;
    cfg.numAttrs = 1;
    if (cfg.dynamicSmemBytes > 48 * 1024)
      if (int rc = allow_shared()) return rc;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, k_select, p);
  if (err != cudaSuccess) return akv_cuda_fail(err, what);
  return AKV_OK;
}
